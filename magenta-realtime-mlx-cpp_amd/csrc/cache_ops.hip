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
      // the running sum of the group's key i, by lane i < 8
      const int key = base + lane_key(g, i & 7), slot = (fresh ? len : 0) + key;
      float sum = 0.f;
      if (i < 8 && key < end) sum = row0 > 0 ? score_out[slot] : fresh || score == nullptr ? 0.f : score[slot];
      int kpos[8];
      if (a.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int kj = min(base + lane_key(g, j), end - 1);
          kpos[j] = fresh ? first + kj : pos != nullptr ? pos[kj] : kj;
        }
      }
      float w[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        if (row0 + t * 16 >= R) continue;
        const f32x4_t x = F::scores(kf[0], q[t]), y = F::scores(kf[1], q[t]);
        const float s[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float z = 0.f;
          if (a.bias != nullptr)
            z = a.bias[(size_t)head[t] * a.buckets + min(max(first + tok[t] - kpos[j], 0), a.buckets - 1)];
          z = __builtin_amdgcn_exp2f((fmaf(s[j], a.scale, z) - lse[t]) * kLog2e);
          w[j] += on[t] && !(fresh && base + lane_key(g, j) > tok[t]) ? z : 0.f;
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
// For each (sequence, head): the `keep` best entries by radix selection on ordered keys,
// then the kept entries at or above the new length go to the evicted slots below it, in
// order: no row is read that another move writes, so the moves need no order among
// themselves.  Ranks come from ballots over consecutive slots, so the result is the same
// on every run.  Short caches (k_evict_short): one wave holds a head's keys in registers
// and finds the threshold by ballots, a bit at a time, with no barrier.  Long ones
// (k_evict_select): a block a head, 11 bits a pass through LDS histograms until the keys
// that are left fit LDS.

constexpr uint32_t kLowest = 0x007fffffu;  // of -inf; a NaN counts as that
constexpr uint32_t kFixed = 0xffffffffu;   // entries that stay

struct EvictK {
  void *k, *v;
  const int *length, *pos, *next_pos;
  const float* score;
  float* score_out;
  int *pos_out, *length_out;
  uint32_t* keys;               // (rows * kv_heads, capacity): k_evict_select
  int *holes, *movers, *count;  // (rows * kv_heads, list), (rows * kv_heads): for k_evict_move, or nullptr
  int64_t c_row, c_head, c_slot;
  int capacity, kv_heads, keep, recent, sinks, list, row_bytes, esz;
};

__device__ __forceinline__ uint32_t evict_key(int p, float f, int64_t recent_from, int sinks) {
  if (p >= recent_from || p < sinks) return kFixed;
  return f != f ? kLowest : float_key(f + 0.f);  // -0 counts as 0
}

__device__ __forceinline__ void move_row(const EvictK& a, int64_t base, int from, int to, int piece) {
  const int64_t e = a.c_slot * a.esz;
  char* kp = static_cast<char*>(a.k) + base + piece * 16;
  char* vp = static_cast<char*>(a.v) + base + piece * 16;
  const uint4 x = ld_g16(kp + from * e), y = ld_g16(vp + from * e);
  *reinterpret_cast<uint4*>(kp + to * e) = x;
  *reinterpret_cast<uint4*>(vp + to * e) = y;
}

constexpr int kShortSlots = 2048;  // capacity up to which k_evict_short serves
constexpr int kShortList = 1024;   // rows that it moves itself

// Four waves load and move; the first finds the threshold from KPT keys a lane, slot 64 t
// + lane in key t, so that ballots are in slot order.
template <int KPT>
__global__ __launch_bounds__(256) void k_evict_short(const EvictK a) {
  constexpr int W = 4, PER = (KPT + W - 1) / W;
  const int bg = blockIdx.x, b = bg / a.kv_heads, kvh = bg - b * a.kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t at = (int64_t)bg * a.capacity;
  __shared__ uint32_t keys[KPT * 64];
  __shared__ uint32_t few[64];
  __shared__ uint64_t kept_of[KPT];
  __shared__ int hole_base[KPT + 1], mover_base[KPT];
  __shared__ int hole_at[kShortList], mover_at[kShortList];
  float f[PER];
  int p[PER];
#pragma unroll
  for (int z = 0; z < PER; ++z) {
    const int j = (z * W + wid) * 64 + lane;
    f[z] = j < a.capacity ? ld_g(a.score + at + j) : 0.f;
    p[z] = j < a.capacity ? ld_g(a.pos + at + j) : 0;
  }
  const int len = min(max(a.length[b], 0), a.capacity), m = min(len, a.keep);
  const int64_t recent_from = (int64_t)a.next_pos[b] - a.recent;
  if (kvh == 0 && tid == 0) a.length_out[b] = m;
#pragma unroll
  for (int z = 0; z < PER; ++z) {
    const int t = z * W + wid, j = t * 64 + lane;
    if (t < KPT) keys[j] = j < len ? evict_key(p[z], f[z], recent_from, a.sinks) : 0u;  // 0: no entry's key
  }
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
  if (wid == 0) {
    uint32_t key[KPT];
#pragma unroll
    for (int t = 0; t < KPT; ++t) key[t] = keys[t * 64 + lane];
    // The largest threshold `low` that at least m keys reach, a bit at a time; once no
    // more than 64 keys share the bits found, one key a lane is enough.
    uint32_t low = m < len ? 0 : 1;
    int reach = len, over = 0;  // keys >= low; keys beyond those that share its bits
    int bit = m < len ? 31 : -1;
    for (; bit >= 0; --bit) {
      const uint32_t x = low | (1u << bit);
      int c = 0;
#pragma unroll
      for (int t = 0; t < KPT; ++t) c += __popcll(__ballot(key[t] >= x));
      if (c >= m) low = x, reach = c;
      else over = c;
      if (reach - over <= 64) break;
    }
    if (bit > 0) {
      int n = 0;
#pragma unroll
      for (int t = 0; t < KPT; ++t) {
        const bool in = key[t] != 0 && (key[t] >> bit) == (low >> bit);
        const uint64_t who = __ballot(in);
        if (in) few[n + __popcll(who & below)] = key[t];
        n += __popcll(who);
      }
      __builtin_amdgcn_wave_barrier();
      const uint32_t one = lane < n ? few[lane] : 0u;
      const int beyond = over;
      for (--bit; bit >= 0; --bit) {
        const uint32_t x = low | (1u << bit);
        const int c = beyond + __popcll(__ballot(one >= x));
        if (c >= m) low = x;
        else over = c;
      }
    }
    // Every key above `low` is kept (`over` of them), and the first ties.
    const int ties = m < len ? m - over : 0;
    int seen = 0, holes = 0, movers = 0;
#pragma unroll
    for (int t = 0; t < KPT; ++t) {
      const int j = t * 64 + lane;
      const uint64_t eq = __ballot(key[t] == low);
      const bool k = m < len ? key[t] > low || (key[t] == low && seen + __popcll(eq & below) < ties) : j < len;
      seen += __popcll(eq);
      const uint64_t who = __ballot(k);
      if (lane == 0) kept_of[t] = who, hole_base[t] = holes, mover_base[t] = movers;
      const int inside = min(max(m - t * 64, 0), 64);  // slots of these below m
      const uint64_t head = inside == 64 ? ~0ull : (1ull << inside) - 1;
      holes += inside - __popcll(who & head), movers += __popcll(who & ~head);
    }
    if (lane == 0) hole_base[KPT] = holes;
  }
  __syncthreads();
  int* hl = a.holes != nullptr ? a.holes + (int64_t)bg * a.list : hole_at;
  int* ml = a.holes != nullptr ? a.movers + (int64_t)bg * a.list : mover_at;
#pragma unroll
  for (int z = 0; z < PER; ++z) {
    const int t = z * W + wid, j = t * 64 + lane;
    if (t >= KPT) continue;
    const uint64_t who = kept_of[t];
    const int inside = min(max(m - t * 64, 0), 64);
    const uint64_t head = inside == 64 ? ~0ull : (1ull << inside) - 1;
    const bool k = (who >> lane) & 1;
    if (j < m && k) a.score_out[at + j] = f[z], a.pos_out[at + j] = p[z];
    if (j < m && !k) hl[hole_base[t] + __popcll(~who & head & below)] = j;
    if (j >= m && k) ml[mover_base[t] + __popcll(who & ~head & below)] = j;
  }
  const int total = hole_base[KPT];
  if (a.holes != nullptr) __threadfence_block();
  __syncthreads();
  if (a.count != nullptr) {
    if (tid == 0) a.count[bg] = total;
    for (int x = tid; x < total; x += 256) {
      const int to = hl[x], from = ml[x];
      a.score_out[at + to] = ld_g(a.score + at + from), a.pos_out[at + to] = ld_g(a.pos + at + from);
    }
    return;
  }
  const int64_t base = (b * a.c_row + kvh * a.c_head) * a.esz;
  const int pieces = a.row_bytes / 16;
#pragma unroll 2
  for (int x = tid; x < total * pieces; x += 256) {
    const int r = x / pieces, piece = x - r * pieces, from = ml[r], to = hl[r];
    move_row(a, base, from, to, piece);
    if (piece == 0) a.score_out[at + to] = ld_g(a.score + at + from), a.pos_out[at + to] = ld_g(a.pos + at + from);
  }
}

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64, kSelBatch = 16;
constexpr int kDigit = 11, kBins = 1 << kDigit, kFew = 8192;  // bins of a pass; keys that LDS takes for the rest

__global__ __launch_bounds__(kSelThreads) void k_evict_select(const EvictK a) {
  constexpr int W = kSelWaves, kRep = 4;
  const int bg = blockIdx.x, b = bg / a.kv_heads, kvh = bg - b * a.kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int len = min(max(a.length[b], 0), a.capacity), m = min(len, a.keep);
  const int64_t at = (int64_t)bg * a.capacity;
  const float* score = a.score + at;
  const int* pos = a.pos + at;
  float* score_out = a.score_out + at;
  int* pos_out = a.pos_out + at;
  uint32_t* keys = a.keys + at;
  if (kvh == 0 && tid == 0) a.length_out[b] = m;
  if (m == len) {
    for (int j = tid; j < len; j += kSelThreads) score_out[j] = score[j], pos_out[j] = pos[j];
    if (tid == 0) a.count[bg] = 0;
    return;
  }
  const int64_t recent_from = (int64_t)a.next_pos[b] - a.recent;
  // Wave w owns slots [w run, (w + 1) run), 64 a turn.  f(slot, key, in use) in slot
  // order, a batch of keys loaded ahead; only the owner reads what it wrote.
  const int turns = (len + 64 * W - 1) / (64 * W), lo = wid * turns * 64 + lane;
  auto each = [&](auto&& f) {
    for (int t0 = 0; t0 < turns; t0 += kSelBatch) {
      uint32_t k[kSelBatch];
#pragma unroll
      for (int t = 0; t < kSelBatch; ++t) {
        const int j = lo + (t0 + t) * 64;
        k[t] = t0 + t < turns && j < len ? ld_g(keys + j) : 0u;
      }
#pragma unroll
      for (int t = 0; t < kSelBatch; ++t) {
        const int j = lo + (t0 + t) * 64;
        if (t0 + t < turns) f(j, k[t], j < len);
      }
    }
  };

  __shared__ uint32_t hist[kBins * kRep];  // then the few keys that are left
  __shared__ uint32_t total_of[W];
  __shared__ uint32_t picked[4];           // digit, of its keys how many are kept, how many there are; the few's count
  __shared__ int tally[3][W];
  uint32_t prefix = 0, mask = 0, want = m;  // of the keys with this prefix, `want` are kept
  // Picks the digit at `shift` from the histogram: thread t holds bins 2 t, 2 t + 1, and
  // counts from the top.
  auto pick = [&](int shift, int bits) {
    __syncthreads();
    uint32_t c[2] = {0, 0};
#pragma unroll
    for (int r = 0; r < kRep; ++r) {
      c[0] += hist[(2 * tid) * kRep + ((r + tid) & (kRep - 1))];
      c[1] += hist[(2 * tid + 1) * kRep + ((r + tid) & (kRep - 1))];
    }
    uint32_t above = c[0] + c[1];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t x = __shfl_down(above, o, 64);
      if (lane + o < 64) above += x;
    }
    if (lane == 0) total_of[wid] = above;
    __syncthreads();
    above -= c[0] + c[1];
    for (int w = wid + 1; w < W; ++w) above += total_of[w];
#pragma unroll
    for (int j = 1; j >= 0; --j) {
      if (above < want && want <= above + c[j]) picked[0] = 2 * tid + j, picked[1] = want - above, picked[2] = c[j];
      above += c[j];
    }
    __syncthreads();
    prefix |= picked[0] << shift;
    mask |= ((1u << bits) - 1) << shift;
    want = picked[1];
  };
  auto clear = [&] {
    for (int x = tid; x < kBins * kRep; x += kSelThreads) hist[x] = 0;
    __syncthreads();
  };
  auto count = [&](uint32_t digit) { atomicAdd(&hist[digit * kRep + (lane & (kRep - 1))], 1u); };
  clear();
  for (int t0 = 0; t0 < turns; t0 += kSelBatch) {
    float f[kSelBatch];
    int p[kSelBatch];
#pragma unroll
    for (int t = 0; t < kSelBatch; ++t) {
      const int j = lo + (t0 + t) * 64;
      const bool in = t0 + t < turns && j < len;
      f[t] = in ? ld_g(score + j) : 0.f;
      p[t] = in ? ld_g(pos + j) : 0;
    }
#pragma unroll
    for (int t = 0; t < kSelBatch; ++t) {
      const int j = lo + (t0 + t) * 64;
      if (t0 + t >= turns || j >= len) continue;
      const uint32_t key = evict_key(p[t], f[t], recent_from, a.sinks);
      keys[j] = key;
      if (j < m) score_out[j] = f[t], pos_out[j] = p[t];  // k_evict_move overwrites the evicted ones
      count(key >> 21);
    }
  }
  pick(21, kDigit);
  int shift = 21;
  while (shift > 0 && picked[2] > kFew) {  // crowded: another pass over all keys
    const int bits = shift > kDigit ? kDigit : shift;
    __syncthreads();  // picked has been read
    clear();
    each([&](int, uint32_t key, bool in) {
      if (in && (key & mask) == prefix) count((key >> (shift - bits)) & ((1u << bits) - 1));
    });
    shift -= bits;
    pick(shift, bits);
  }
  if (shift > 0) {  // the rest from LDS, a bit at a time
    if (tid == 0) picked[3] = 0;
    __syncthreads();
    each([&](int, uint32_t key, bool in) {
      const bool mine = in && (key & mask) == prefix;
      const uint64_t who = __ballot(mine);
      uint32_t first = 0;
      if (who != 0 && lane == 0) first = atomicAdd(&picked[3], (uint32_t)__popcll(who));
      first = __builtin_amdgcn_readfirstlane(first);
      if (mine) hist[first + __popcll(who & ((1ull << lane) - 1))] = key;
    });
    __syncthreads();
    const int n = picked[3];
    uint32_t k[kFew / kSelThreads];
#pragma unroll
    for (int z = 0; z < kFew / kSelThreads; ++z) k[z] = tid + z * kSelThreads < n ? hist[tid + z * kSelThreads] : 0u;
    for (int bit = shift - 1; bit >= 0; --bit) {
      const uint32_t x = prefix | (1u << bit);
      int c = 0;
#pragma unroll
      for (int z = 0; z < kFew / kSelThreads; ++z) c += __popcll(__ballot(k[z] >= x && k[z] >> bit == x >> bit));
      if (lane == 0) tally[bit & 1][wid] = c;
      __syncthreads();
      int sum = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) sum += tally[bit & 1][w];
      if (sum >= (int)want) prefix = x;
      else want -= sum;
    }
    __syncthreads();
  }
  // Kept: keys above prefix, and the first `want` slots with it.
  int equal = 0;
  each([&](int, uint32_t key, bool in) { equal += __popcll(__ballot(in && key == prefix)); });
  if (lane == 0) tally[0][wid] = equal;
  __syncthreads();
  int ties = 0;
  for (int w = 0; w < wid; ++w) ties += tally[0][w];
  const uint64_t below = (1ull << lane) - 1;
  auto kept_of = [&](uint32_t key, bool in, int& seen) -> bool {
    const uint64_t eq = __ballot(in && key == prefix);
    const bool k = in && (key > prefix || (key == prefix && seen + __popcll(eq & below) < (int)want));
    seen += __popcll(eq);
    return k;
  };
  int seen = ties, holes = 0, movers = 0;
  each([&](int j, uint32_t key, bool in) {
    const bool k = kept_of(key, in, seen);
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
  int* hl = a.holes + (int64_t)bg * a.list;
  int* ml = a.movers + (int64_t)bg * a.list;
  seen = ties;
  each([&](int j, uint32_t key, bool in) {
    const bool k = kept_of(key, in, seen);
    const uint64_t h = __ballot(j < m && !k), v = __ballot(j >= m && k);
    if (j < m && !k) hl[hole + __popcll(h & below)] = j;
    if (j >= m && k) ml[mover + __popcll(v & below)] = j;
    hole += __popcll(h), mover += __popcll(v);
  });
  if (tid == 0) a.count[bg] = total;
}

// Rows of the lists, `blocks` blocks a (sequence, head); with `entries`, their scores and
// positions too.
__global__ __launch_bounds__(256) void k_evict_move(const EvictK a, int blocks, bool entries) {
  const int bg = blockIdx.x / blocks, part = blockIdx.x - bg * blocks, b = bg / a.kv_heads, kvh = bg - b * a.kv_heads;
  const int pieces = a.row_bytes / 16;
  const int64_t total = (int64_t)a.count[bg] * pieces, base = (b * a.c_row + kvh * a.c_head) * a.esz;
  const int64_t at = (int64_t)bg * a.capacity;
  const int* hl = a.holes + (int64_t)bg * a.list;
  const int* ml = a.movers + (int64_t)bg * a.list;
  for (int64_t x = part * 256 + threadIdx.x; x < total; x += (int64_t)blocks * 256) {
    const int r = (int)(x / pieces), piece = (int)(x - (int64_t)r * pieces), from = ml[r], to = hl[r];
    move_row(a, base, from, to, piece);
    if (entries && piece == 0) a.score_out[at + to] = a.score[at + from], a.pos_out[at + to] = a.pos[at + from];
  }
}

// Most rows that a head can move; whether k_evict_short serves, and moves them itself.
int most_moves(const KvCache& c, int keep) { return std::max(0, std::min(keep, c.capacity - keep)); }
bool is_short(const KvCache& c) { return c.capacity <= kShortSlots; }
bool moves_within(const KvCache& c, int keep) {
  return is_short(c) && (size_t)most_moves(c, keep) * c.d * dtype_size(c.dt) <= 16 * 1024;
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
  return heads * (2 * (size_t)most_moves(c, keep) + 1 + (is_short(c) ? 0 : (size_t)c.capacity)) * 4;
}

void cache_evict(const KvCache& c, const EvictArgs& t, void* ws, hipStream_t s) {
  EvictK a{};
  a.k = c.k, a.v = c.v, a.length = c.length, a.pos = c.pos, a.next_pos = c.next_pos, a.score = c.score;
  a.score_out = t.score_out, a.pos_out = t.pos_out, a.length_out = t.length_out;
  a.c_row = c.row_stride, a.c_head = c.head_stride, a.c_slot = c.slot_stride;
  a.capacity = c.capacity, a.kv_heads = c.kv_heads, a.keep = t.keep, a.recent = t.recent, a.sinks = t.sinks;
  a.esz = (int)dtype_size(c.dt), a.row_bytes = c.d * a.esz, a.list = most_moves(c, t.keep);
  const int heads = c.rows * c.kv_heads;
  if (!moves_within(c, t.keep)) {
    a.holes = static_cast<int*>(ws);
    a.movers = a.holes + (size_t)heads * a.list;
    a.count = a.movers + (size_t)heads * a.list;
    a.keys = reinterpret_cast<uint32_t*>(a.count + heads);
  }
  if (c.capacity <= 8 * 64) hipLaunchKernelGGL(k_evict_short<8>, dim3(heads), dim3(256), 0, s, a);
  else if (c.capacity <= 18 * 64) hipLaunchKernelGGL(k_evict_short<18>, dim3(heads), dim3(256), 0, s, a);
  else if (is_short(c)) hipLaunchKernelGGL(k_evict_short<32>, dim3(heads), dim3(256), 0, s, a);
  else hipLaunchKernelGGL(k_evict_select, dim3(heads), dim3(kSelThreads), 0, s, a);
  MRT_HIP_CHECK(hipGetLastError());
  if (a.holes != nullptr && a.list > 0) {
    const int64_t pieces = (int64_t)a.list * (a.row_bytes / 16);
    const int blocks = (int)std::max<int64_t>(1, std::min<int64_t>((pieces + 1023) / 1024, 8192 / heads));
    hipLaunchKernelGGL(k_evict_move, dim3(blocks * heads), dim3(256), 0, s, a, blocks, !is_short(c));
    MRT_HIP_CHECK(hipGetLastError());
  }
}

}  // namespace mrt
