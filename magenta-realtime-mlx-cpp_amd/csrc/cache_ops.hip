// Commit of an accepted path into a cache, and eviction by accumulated attention
// weight.
#include <algorithm>

#include "attn_frag.hpp"
#include "kv_cache.hpp"
#include "mfma_ring.hpp"

namespace mrt {
namespace {

// ---- commit ---------------------------------------------------------------------
//
// score'_j = score_j + sum over accepted tokens i and the query heads of the KV head of
// exp(scale q_i . k_j + bias - lse_i), for the entries at or before the token.  Reads
// every key once (values not at all): 32 keys a step as attention does (attn_frag.hpp),
// each lane summing its eight keys over row tiles, 16 lanes a row tile at the end.  The
// rows (token, head) beyond 16 NR take another turn over the keys.  Accepted rows are
// copied by the first block of a head; all keys they are scored against come from
// k_new, so that no block waits for another.

constexpr int kCommitWaves = 4;

struct CommitK {
  const void *k_new, *v_new, *q;
  void *k, *v;
  const int *accepted, *length, *next_pos;
  int* pos;
  const float *lse, *bias, *score;
  float* score_out;
  int *length_out, *next_out;
  int64_t q_row, q_node, q_head, kn_row, kn_node, kn_head, vn_row, vn_node, vn_head;
  int64_t c_row, c_head, c_slot, accepted_stride;
  int capacity, kv_heads, heads, nodes, accepted_n, D, buckets, splits, split_steps;
  float scale;
};

template <typename T, int DP, int NR>
__global__ __launch_bounds__(64 * kCommitWaves) void k_commit(const CommitK a) {
  using F = AttnFrag<T, DP>;
  constexpr int KC = F::KC;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4, D = a.D;
  const int bg = blockIdx.x / a.splits, split = blockIdx.x - bg * a.splits;
  const int b = bg / a.kv_heads, kvh = bg - b * a.kv_heads, nh = a.heads / a.kv_heads;
  const int len = min(max(a.length[b], 0), a.capacity);

  // The accepted prefix: ascending nodes that the cache has room for.
  __shared__ int acc[kMaxNodes];
  const int mine = lane < a.accepted_n ? a.accepted[b * a.accepted_stride + lane] : -1;
  int before = __shfl_up(mine, 1, 64);
  if (lane == 0) before = -1;
  const uint64_t bad = ~__ballot(mine > before && mine < a.nodes && len + lane < a.capacity);
  const int n = bad == 0 ? 64 : __ffsll((unsigned long long)bad) - 1;
  if (wid == 0) acc[lane] = lane < n ? mine : 0;
  __syncthreads();
  const int first = a.next_pos != nullptr ? a.next_pos[b] : len;
  const T* kn = static_cast<const T*>(a.k_new) + b * a.kn_row + kvh * a.kn_head;
  T* kc = static_cast<T*>(a.k) + b * a.c_row + kvh * a.c_head;
  int* pos = a.pos == nullptr ? nullptr : a.pos + (size_t)bg * a.capacity;

  if (split == 0) {
    const T* vn = static_cast<const T*>(a.v_new) + b * a.vn_row + kvh * a.vn_head;
    T* vc = static_cast<T*>(a.v) + b * a.c_row + kvh * a.c_head;
    constexpr int kElt = 16 / sizeof(T);
    const int pieces = D / kElt;
    for (int x = tid; x < n * pieces; x += 64 * kCommitWaves) {
      const int r = x / pieces, d = (x - r * pieces) * kElt;
      const uint4 kv = ld_g16(kn + acc[r] * a.kn_node + d), vv = ld_g16(vn + acc[r] * a.vn_node + d);
      *reinterpret_cast<uint4*>(kc + (int64_t)(len + r) * a.c_slot + d) = kv;
      *reinterpret_cast<uint4*>(vc + (int64_t)(len + r) * a.c_slot + d) = vv;
    }
    if (pos != nullptr && tid < n) pos[len + tid] = first + tid;
    if (kvh == 0 && tid == 0) {
      a.length_out[b] = len + n;
      if (a.next_out != nullptr) a.next_out[b] = first + n;
    }
  }
  if (a.q == nullptr) return;

  const int old_steps = (len + kStepKeys - 1) / kStepKeys, steps = old_steps + (n + kStepKeys - 1) / kStepKeys;
  const int s0 = split * a.split_steps, s1 = min(steps, s0 + a.split_steps);
  const int R = n * nh;
  const float* score = a.score == nullptr ? nullptr : a.score + (size_t)bg * a.capacity;
  float* score_out = a.score_out + (size_t)bg * a.capacity;
  if (R == 0) {
    if (score != nullptr && score != score_out)
      for (int j = s0 * kStepKeys + tid; j < min(len, s1 * kStepKeys); j += 64 * kCommitWaves) score_out[j] = score[j];
    return;
  }
  for (int row0 = 0; row0 < R; row0 += 16 * NR) {
    uint4 q[NR][KC];
    float lse[NR];
    int tok[NR], head[NR];
    bool on[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      const int row = row0 + t * 16 + i, r = min(row, R - 1);
      tok[t] = r / nh, head[t] = kvh * nh + r - tok[t] * nh;
      F::load_row(static_cast<const T*>(a.q) + b * a.q_row + acc[tok[t]] * a.q_node + head[t] * a.q_head, g, D, q[t]);
      lse[t] = a.lse[((size_t)b * a.nodes + acc[tok[t]]) * a.heads + head[t]];
      on[t] = row < R && lse[t] > -INFINITY;
    }
    for (int st = s0 + wid; st < s1; st += kCommitWaves) {
      const bool fresh = st >= old_steps;
      const int base = (fresh ? st - old_steps : st) * kStepKeys, end = fresh ? n : len;
      uint4 kf[2][KC];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = min(base + step_key(i, h), end - 1);
        F::load_row(fresh ? kn + acc[key] * a.kn_node : kc + (int64_t)key * a.c_slot, g, D, kf[h]);
      }
      // the running sum of key base + 8 g + i, by lane i < 8
      const int key = base + 8 * g + (i & 7), slot = (fresh ? len : 0) + key;
      float sum = 0.f;
      if (i < 8 && key < end) sum = row0 > 0 ? score_out[slot] : fresh || score == nullptr ? 0.f : score[slot];
      int kpos[8];
      if (a.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int kj = min(base + 8 * g + j, end - 1);
          kpos[j] = fresh ? first + kj : pos != nullptr ? pos[kj] : kj;
        }
      }
      float w[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        const f32x4_t x = F::scores(kf[0], q[t]), y = F::scores(kf[1], q[t]);
        const float s[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float z = 0.f;
          if (a.bias != nullptr)
            z = a.bias[(size_t)head[t] * a.buckets + min(max(first + tok[t] - kpos[j], 0), a.buckets - 1)];
          z = __builtin_amdgcn_exp2f((fmaf(s[j], a.scale, z) - lse[t]) * kLog2e);
          w[j] += on[t] && !(fresh && base + 8 * g + j > tok[t]) ? z : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = sum_in_group(w[j]);
        sum += (i & 7) == j ? w[j] : 0.f;
      }
      if (i < 8 && key < end) score_out[slot] = sum;
    }
  }
}

template <typename T, int DP>
void launch_commit(const CommitK& a, int rows, int nr, hipStream_t s) {
  const dim3 grid(rows * a.kv_heads * a.splits), block(64 * kCommitWaves);
  if (nr == 1) {
    hipLaunchKernelGGL((k_commit<T, DP, 1>), grid, block, 0, s, a);
    return;
  }
  constexpr int most = DP == 256 || (sizeof(T) == 4 && DP == 128) ? 2 : 4;
  hipLaunchKernelGGL((k_commit<T, DP, most>), grid, block, 0, s, a);
}

// ---- eviction -------------------------------------------------------------------
//
// A block a (sequence, head) finds the `keep` best of its entries by radix selection on
// ordered keys (8 bits a pass, highest first), then moves the kept entries that lie at
// or above the new length into the evicted slots below it, in order: no row is read
// that another move writes, so the moves of a head need no order among themselves.
// Each wave owns a run of consecutive slots, so that ranks are a count per wave, a sum
// over the waves before and a ballot, and the result is the same on every run.

constexpr uint32_t kLowest = 0x007fffffu;  // of -inf; a NaN counts as that
constexpr uint32_t kFixed = 0xffffffffu;   // entries that stay

struct EvictK {
  void *k, *v;
  const int *length, *pos, *next_pos;
  const float* score;
  float* score_out;
  int *pos_out, *length_out;
  int *holes, *movers, *count;  // (rows * kv_heads, list), (rows * kv_heads): for k_evict_move, or nullptr
  int64_t c_row, c_head, c_slot;
  int capacity, kv_heads, keep, recent, sinks, list, row_bytes, esz;
};

__device__ __forceinline__ void move_row(const EvictK& a, int64_t base, int from, int to, int piece) {
  const int64_t e = a.c_slot * a.esz;
  char* kp = static_cast<char*>(a.k) + base + piece * 16;
  char* vp = static_cast<char*>(a.v) + base + piece * 16;
  const uint4 x = ld_g16(kp + from * e), y = ld_g16(vp + from * e);
  *reinterpret_cast<uint4*>(kp + to * e) = x;
  *reinterpret_cast<uint4*>(vp + to * e) = y;
}

// Threads a block, keys a thread held in registers (0: read again in every pass).
template <int THREADS, int KPT>
__global__ __launch_bounds__(THREADS) void k_evict_select(const EvictK a) {
  constexpr int W = THREADS / 64, kRep = 16;
  const int bg = blockIdx.x, b = bg / a.kv_heads, kvh = bg - b * a.kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int len = min(max(a.length[b], 0), a.capacity), m = min(len, a.keep);
  const int64_t at = (int64_t)bg * a.capacity;
  const float* score = a.score + at;
  const int* pos = a.pos + at;
  float* score_out = a.score_out + at;
  int* pos_out = a.pos_out + at;
  if (kvh == 0 && tid == 0) a.length_out[b] = m;
  if (a.count != nullptr && tid == 0) a.count[bg] = 0;
  if (m == len) {
    for (int j = tid; j < len; j += THREADS) score_out[j] = score[j], pos_out[j] = pos[j];
    return;
  }
  const int64_t recent_from = (int64_t)a.next_pos[b] - a.recent;
  // wave w owns slots [w run, (w + 1) run), 64 a turn
  const int turns = (len + 64 * W - 1) / (64 * W), run = turns * 64;
  const int lo = wid * run + lane;
  auto key_at = [&](int t) -> uint32_t {
    const int j = lo + t * 64;
    if (j >= len) return 0u;
    const int p = ld_g(pos + j);
    const float f = ld_g(score + j);
    if (p >= recent_from || p < a.sinks) return kFixed;
    return f != f ? kLowest : float_key(f + 0.f);  // -0 counts as 0
  };
  constexpr int kHeld = KPT > 0 ? KPT : 1;
  uint32_t held[kHeld];
  if constexpr (KPT > 0) {
#pragma unroll
    for (int t = 0; t < KPT; ++t) held[t] = t < turns ? key_at(t) : 0u;
  }
  auto each = [&](auto&& f) {  // f(turn, key) in slot order
    if constexpr (KPT > 0) {
#pragma unroll
      for (int t = 0; t < KPT; ++t)
        if (t < turns) f(t, held[t]);
    } else {
      for (int t = 0; t < turns; ++t) f(t, key_at(t));
    }
  };

  __shared__ uint32_t hist[256 * kRep];
  __shared__ uint32_t bins[256];
  __shared__ uint32_t picked[2];
  __shared__ int tally[3][W];
  uint32_t prefix = 0, mask = 0, want = m;  // of the keys with this prefix, `want` are kept
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int x = tid; x < 256 * kRep; x += THREADS) hist[x] = 0;
    __syncthreads();
    each([&](int t, uint32_t key) {
      if (lo + t * 64 < len && (key & mask) == prefix) atomicAdd(&hist[((key >> shift) & 255) * kRep + (lane & (kRep - 1))], 1u);
    });
    __syncthreads();
    for (int x = tid; x < 256; x += THREADS) {
      uint32_t c = 0;
#pragma unroll
      for (int r = 0; r < kRep; ++r) c += hist[x * kRep + ((r + x) & (kRep - 1))];
      bins[x] = c;
    }
    __syncthreads();
    if (wid == 0) {  // lane l: bins 4 l .. 4 l + 3; counts from the top
      const uint32_t c0 = bins[4 * lane], c1 = bins[4 * lane + 1], c2 = bins[4 * lane + 2], c3 = bins[4 * lane + 3];
      uint32_t above = c0 + c1 + c2 + c3;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_down(above, o, 64);
        if (lane + o < 64) above += x;
      }
      above -= c0 + c1 + c2 + c3;  // in the lanes above
      const uint32_t c[4] = {c0, c1, c2, c3};
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        if (above < want && want <= above + c[j]) picked[0] = 4 * lane + j, picked[1] = want - above;
        above += c[j];
      }
    }
    __syncthreads();
    prefix |= picked[0] << shift;
    mask |= 255u << shift;
    want = picked[1];
  }
  // Kept: keys above prefix, and the first `want` slots with it.
  int equal = 0;
  each([&](int t, uint32_t key) { equal += __popcll(__ballot(lo + t * 64 < len && key == prefix)); });
  if (lane == 0) tally[0][wid] = equal;
  __syncthreads();
  int ties = 0;
  for (int w = 0; w < wid; ++w) ties += tally[0][w];
  const uint64_t below = (1ull << lane) - 1;
  auto kept_of = [&](int t, uint32_t key, int& seen) -> bool {
    const uint64_t eq = __ballot(lo + t * 64 < len && key == prefix);
    const bool k = lo + t * 64 < len && (key > prefix || (key == prefix && seen + __popcll(eq & below) < (int)want));
    seen += __popcll(eq);
    return k;
  };
  int seen = ties, holes = 0, movers = 0;
  each([&](int t, uint32_t key) {
    const bool k = kept_of(t, key, seen);
    const int j = lo + t * 64;
    holes += __popcll(__ballot(j < m && !k));
    movers += __popcll(__ballot(j >= m && k));
  });
  if (lane == 0) tally[1][wid] = holes, tally[2][wid] = movers;
  __syncthreads();
  int hole = 0, mover = 0, total = 0;
  for (int w = 0; w < W; ++w) {
    if (w < wid) hole += tally[1][w], mover += tally[2][w];
    total += tally[1][w];
  }
  extern __shared__ int lists[];  // holes, movers, where they are not in memory
  int* hl = a.holes != nullptr ? a.holes + (int64_t)bg * a.list : lists;
  int* ml = a.holes != nullptr ? a.movers + (int64_t)bg * a.list : lists + a.list;
  seen = ties;
  each([&](int t, uint32_t key) {
    const bool k = kept_of(t, key, seen);
    const int j = lo + t * 64;
    const uint64_t h = __ballot(j < m && !k), v = __ballot(j >= m && k);
    if (j < m && !k) hl[hole + __popcll(h & below)] = j;
    if (j >= m && k) ml[mover + __popcll(v & below)] = j;
    hole += __popcll(h), mover += __popcll(v);
    if (j < m && k) score_out[j] = score[j], pos_out[j] = pos[j];
  });
  if (a.holes != nullptr) __threadfence_block();
  __syncthreads();
  for (int x = tid; x < total; x += THREADS) {
    const int to = hl[x], from = ml[x];
    score_out[to] = score[from], pos_out[to] = pos[from];
  }
  if (a.count != nullptr) {
    if (tid == 0) a.count[bg] = total;
    return;
  }
  const int64_t base = (b * a.c_row + kvh * a.c_head) * a.esz;
  const int pieces = a.row_bytes / 16;
  for (int x = tid; x < total * pieces; x += THREADS) {
    const int r = x / pieces;
    move_row(a, base, ml[r], hl[r], x - r * pieces);
  }
}

// Rows of the long lists, `blocks` blocks a (sequence, head).
__global__ __launch_bounds__(256) void k_evict_move(const EvictK a, int blocks) {
  const int bg = blockIdx.x / blocks, part = blockIdx.x - bg * blocks, b = bg / a.kv_heads, kvh = bg - b * a.kv_heads, pieces = a.row_bytes / 16;
  const int64_t total = (int64_t)a.count[bg] * pieces, base = (b * a.c_row + kvh * a.c_head) * a.esz;
  const int* hl = a.holes + (int64_t)bg * a.list;
  const int* ml = a.movers + (int64_t)bg * a.list;
  for (int64_t x = part * 256 + threadIdx.x; x < total; x += (int64_t)blocks * 256) {
    const int r = (int)(x / pieces);
    move_row(a, base, ml[r], hl[r], (int)(x - (int64_t)r * pieces));
  }
}

// Most rows that a head can move, and whether its block moves them itself.
int most_moves(const KvCache& c, int keep) { return std::max(0, std::min(keep, c.capacity - keep)); }
bool moves_within(const KvCache& c, int keep) {
  return (size_t)most_moves(c, keep) * c.d * dtype_size(c.dt) <= 64 * 1024;
}

}  // namespace

void cache_commit(const KvCache& c, const CommitArgs& t, hipStream_t s) {
  CommitK a{};
  a.k_new = t.k_new.p, a.v_new = t.v_new.p, a.q = t.q.p, a.k = c.k, a.v = c.v;
  a.accepted = t.accepted, a.length = c.length, a.next_pos = c.pos != nullptr ? c.next_pos : nullptr, a.pos = c.pos;
  a.lse = t.lse, a.bias = t.bias, a.score = c.score, a.score_out = t.score_out;
  a.length_out = t.length_out, a.next_out = c.pos != nullptr ? t.next_out : nullptr;
  a.q_row = t.q.row_stride, a.q_node = t.q.node_stride, a.q_head = t.q.head_stride;
  a.kn_row = t.k_new.row_stride, a.kn_node = t.k_new.node_stride, a.kn_head = t.k_new.head_stride;
  a.vn_row = t.v_new.row_stride, a.vn_node = t.v_new.node_stride, a.vn_head = t.v_new.head_stride;
  a.c_row = c.row_stride, a.c_head = c.head_stride, a.c_slot = c.slot_stride, a.accepted_stride = t.accepted_stride;
  a.capacity = c.capacity, a.kv_heads = c.kv_heads, a.heads = t.heads, a.nodes = t.nodes, a.accepted_n = t.accepted_n;
  a.D = c.d, a.buckets = t.buckets, a.scale = t.scale;
  a.splits = 1, a.split_steps = 1 << 30;
  if (t.q.p != nullptr) {
    const int steps = (c.capacity + kStepKeys - 1) / kStepKeys + (t.accepted_n + kStepKeys - 1) / kStepKeys;
    const int want = std::max(1, 2048 / std::max(1, c.rows * c.kv_heads));
    a.split_steps = std::max(2 * kCommitWaves, (steps + want - 1) / want);
    a.splits = (steps + a.split_steps - 1) / a.split_steps;
  }
  const int nr = t.q.p == nullptr || t.accepted_n * (t.heads / c.kv_heads) <= 16 ? 1 : 4;
  MRT_DTYPE_DISPATCH(c.dt, {
    if (c.d <= 32) launch_commit<T, 32>(a, c.rows, nr, s);
    else if (c.d <= 64) launch_commit<T, 64>(a, c.rows, nr, s);
    else if (c.d <= 128) launch_commit<T, 128>(a, c.rows, nr, s);
    else launch_commit<T, 256>(a, c.rows, nr, s);
  });
  MRT_HIP_CHECK(hipGetLastError());
}

size_t cache_evict_workspace(const KvCache& c, int keep) {
  if (moves_within(c, keep)) return 0;
  const size_t heads = (size_t)c.rows * c.kv_heads;
  return heads * (2 * (size_t)most_moves(c, keep) + 1) * 4;
}

void cache_evict(const KvCache& c, const EvictArgs& t, void* ws, hipStream_t s) {
  EvictK a{};
  a.k = c.k, a.v = c.v, a.length = c.length, a.pos = c.pos, a.next_pos = c.next_pos, a.score = c.score;
  a.score_out = t.score_out, a.pos_out = t.pos_out, a.length_out = t.length_out;
  a.c_row = c.row_stride, a.c_head = c.head_stride, a.c_slot = c.slot_stride;
  a.capacity = c.capacity, a.kv_heads = c.kv_heads, a.keep = t.keep, a.recent = t.recent, a.sinks = t.sinks;
  a.esz = (int)dtype_size(c.dt), a.row_bytes = c.d * a.esz, a.list = most_moves(c, t.keep);
  const int heads = c.rows * c.kv_heads;
  size_t lds = (size_t)a.list * 8;
  if (!moves_within(c, t.keep)) {
    a.holes = static_cast<int*>(ws);
    a.movers = a.holes + (size_t)heads * a.list;
    a.count = a.movers + (size_t)heads * a.list;
    lds = 0;
  }
  if (c.capacity <= 256 * 8) hipLaunchKernelGGL((k_evict_select<256, 8>), dim3(heads), dim3(256), lds, s, a);
  else if (c.capacity <= 1024 * 16) hipLaunchKernelGGL((k_evict_select<1024, 16>), dim3(heads), dim3(1024), lds, s, a);
  else if (c.capacity <= 1024 * 72) hipLaunchKernelGGL((k_evict_select<1024, 72>), dim3(heads), dim3(1024), lds, s, a);
  else hipLaunchKernelGGL((k_evict_select<1024, 0>), dim3(heads), dim3(1024), lds, s, a);
  MRT_HIP_CHECK(hipGetLastError());
  if (a.holes != nullptr) {
    const int64_t pieces = (int64_t)a.list * (a.row_bytes / 16);
    const int blocks = (int)std::max<int64_t>(1, std::min<int64_t>((pieces + 1023) / 1024, 8192 / heads));
    hipLaunchKernelGGL(k_evict_move, dim3(blocks * heads), dim3(256), 0, s, a, blocks);
    MRT_HIP_CHECK(hipGetLastError());
  }
}

}  // namespace mrt
