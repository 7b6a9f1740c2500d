// Commit of an accepted path into a cache, and eviction by accumulated attention
// weight.
#include <algorithm>
#include <utility>

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
// rows (token, head) beyond 16 NR take another turn over the keys.  Query rows wait in LDS,
// as the lanes read them: in registers they cost a third of the waves (65 us instead of
// 62).  Bound by the keys: 5 caches of up to 40001, 8 K/V heads, d 128, fp16 (242 MB) 62 us,
// 3.9 TB/s.  Accepted rows are
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
  if (R == 0) {  // nothing accepted: the scores stay, 0 where there were none
    if (score != score_out)
      for (int j = s0 * kStepKeys + tid; j < min(len, s1 * kStepKeys); j += 64 * kCommitWaves)
        score_out[j] = score == nullptr ? 0.f : score[j];
    return;
  }
  __shared__ uint4 rows[NR][KC][64];  // q, as the lanes read it
  for (int row0 = 0; row0 < R; row0 += 16 * NR) {
    float lse[NR];
    int tok[NR], head[NR];
    bool on[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      const int row = row0 + t * 16 + i, r = min(row, R - 1);
      tok[t] = r / nh, head[t] = kvh * nh + r - tok[t] * nh;
      if (wid == t % kCommitWaves) {
        uint4 x[KC];
        F::load_row(static_cast<const T*>(a.q) + b * a.q_row + acc[tok[t]] * a.q_node + head[t] * a.q_head, g, D, x);
#pragma unroll
        for (int c = 0; c < KC; ++c) rows[t][c][lane] = x[c];
      }
      lse[t] = a.lse[((size_t)b * a.nodes + acc[tok[t]]) * a.heads + head[t]];
      on[t] = row < R && lse[t] != -INFINITY;
    }
    __syncthreads();
    for (int st = s0 + wid; st < s1; st += kCommitWaves) {
      const bool fresh = st >= old_steps;
      const int base = (fresh ? st - old_steps : st) * kStepKeys, end = fresh ? n : len;
      uint4 kf[2][KC];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = min(base + step_key(lane >> 2, h), end - 1);
        F::load_row(fresh ? kn + acc[key] * a.kn_node : kc + (int64_t)key * a.c_slot, lane & 3, D, kf[h]);
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
#pragma unroll
      for (int h = 0; h < 2; ++h) F::spread(kf[h], lane);
      float w[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        if (row0 + t * 16 >= R) continue;
        uint4 q[KC];
#pragma unroll
        for (int c = 0; c < KC; ++c) q[c] = rows[t][c][lane];
        const f32x4_t x = F::scores(kf[0], q), y = F::scores(kf[1], q);
        const float s[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float by = 0.f;
          if (a.bias != nullptr)
            by = a.bias[(size_t)head[t] * a.buckets + bucket(first + tok[t], kpos[j], a.buckets)];
          const float z = __builtin_amdgcn_exp2f((fmaf(s[j], a.scale, by) - lse[t]) * kLog2e);
          const bool masked = by * kLog2e < kNone;  // whatever the key holds
          w[j] += on[t] && !masked && !(fresh && base + lane_key(g, j) > tok[t]) ? z : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = sum_in_group(w[j]);
        sum += (i & 7) == j ? w[j] : 0.f;
      }
      if (i < 8 && key < end) score_out[slot] = sum;
    }
    if (row0 + 16 * NR < R) __syncthreads();  // before `rows` is written again
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
// and finds the threshold by ballots, a bit at a time, with no barrier.  Long ones: a head's
// slots go to several blocks.  k_evict_keys counts each part's keys by their first 10 bits,
// k_evict_collect finds the digit that the threshold has from all parts' counts and
// collects its keys, k_evict_lists finds the other 22 bits from these in two passes, each
// block by itself, and lists what moves: no block waits for another, and keys that are all
// alike only make the collected ones more.
// Bound: 64 x 16 heads from 1056 to 1006 entries, d 64 (43 MB), 19 us, one round of blocks
// with five dependent steps; 4 x 8 heads from 65536 to 32768, d 128 (570 MB), 151 us, of
// which 115 move rows at the rate of a copy and 37 find them (one block a head: 111).

constexpr uint32_t kLowest = 0x007fffffu;  // of -inf; a NaN counts as that
constexpr uint32_t kFixed = 0xffffffffu;   // entries that stay

struct EvictK {
  void *k, *v;
  const int *length, *pos, *next_pos;
  const float* score;
  float* score_out;
  int *pos_out, *length_out;
  int *holes, *movers, *count;  // (rows * kv_heads, list), (rows * kv_heads): for k_evict_move, or nullptr
  uint32_t *keys, *few;         // (rows * kv_heads, capacity): of long caches, and what follows
  uint32_t* hist;               // (rows * kv_heads, parts, kBins1)
  int2* part_of;                // (rows * kv_heads, parts): keys in few, keys of higher digits
  uint2* digit;                 // (rows * kv_heads): of `few`, and how many of these are kept
  int64_t c_row, c_head, c_slot;
  int capacity, kv_heads, keep, recent, sinks, list, row_bytes, esz, parts, part_slots;
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

// Capacity up to which k_evict_short serves (what a wave has registers for): 1024 heads from
// 2048 to 1900 42 us, with the kernels of long caches 57; 32 heads to 1024 23 and 21.
constexpr int kShortSlots = 2048;
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
  const int total = hole_base[KPT];
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
    if (j >= m && k) ml[total - 1 - mover_base[t] - __popcll(who & ~head & below)] = j;
  }
  if (a.holes != nullptr) __threadfence_block();
  __syncthreads();
  if (a.count != nullptr) {
    if (tid == 0) a.count[bg] = total;
    for (int x = tid; x < total; x += 256) {
      const int to = hl[x], from = ml[total - 1 - x];
      a.score_out[at + to] = ld_g(a.score + at + from), a.pos_out[at + to] = ld_g(a.pos + at + from);
    }
    return;
  }
  const int64_t base = (b * a.c_row + kvh * a.c_head) * a.esz;
  const int pieces = a.row_bytes / 16;
#pragma unroll 2
  for (int x = tid; x < total * pieces; x += 256) {
    const int r = x / pieces, piece = x - r * pieces, from = ml[total - 1 - r], to = hl[r];
    move_row(a, base, from, to, piece);
    if (piece == 0) a.score_out[at + to] = ld_g(a.score + at + from), a.pos_out[at + to] = ld_g(a.pos + at + from);
  }
}

constexpr int kSelThreads = 512, kSelWaves = kSelThreads / 64, kSelBatch = 8;
constexpr int kPartSlots = kSelThreads * kSelBatch;  // slots of a part: a multiple of these
constexpr int kMostParts = 32;
constexpr int kBins1 = 1 << 10, kBins2 = 1 << 11;    // digits of 10, 11 and 11 bits

// One more key of `digit`, in one of REP copies of the histogram by lane; lanes that share
// the first active lane's digit count as one.
template <int REP>
__device__ __forceinline__ void count_digit(uint32_t* hist, uint32_t digit, int lane) {
  const uint32_t lead = __builtin_amdgcn_readfirstlane(digit);
  const uint64_t who = __ballot(digit == lead);
  if (digit != lead) atomicAdd(&hist[digit * REP + (lane & (REP - 1))], 1u);
  else if (lane == __ffsll((unsigned long long)who) - 1) atomicAdd(&hist[digit * REP], (uint32_t)__popcll(who));
}

// The digit with which the `want` highest of BINS counted digits end: thread t brings the
// counts of digits PER t .. and counts from the top.  Returns it in `picked`: the digit,
// and how many of its keys are among the `want`.
template <int BINS>
__device__ __forceinline__ void pick_digit(const uint32_t (&c)[BINS / kSelThreads], uint32_t want, uint32_t* total_of,
                                           uint32_t* picked) {
  constexpr int PER = BINS / kSelThreads;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  uint32_t own = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) own += c[j];
  uint32_t above = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t x = __shfl_down(above, o, 64);
    if (lane + o < 64) above += x;
  }
  if (lane == 0) total_of[wid] = above;
  __syncthreads();
  above -= own;
  for (int w = wid + 1; w < kSelWaves; ++w) above += total_of[w];
#pragma unroll
  for (int j = PER - 1; j >= 0; --j) {
    if (above < want && want <= above + c[j]) picked[0] = PER * tid + j, picked[1] = want - above;
    above += c[j];
  }
  __syncthreads();
}

// What a block of the three kernels works on.  Blocks of one head are `heads` apart, so
// that they share an L2 where the heads are a multiple of the XCDs.
struct EvictPart {
  int bg, part, parts, len, m, from, to;  // parts in use; slots [from, to)
  size_t id;
  int64_t at;
};
__device__ __forceinline__ EvictPart evict_part(const EvictK& a) {
  EvictPart e;
  const int heads = gridDim.x / a.parts;
  e.part = blockIdx.x / heads, e.bg = blockIdx.x - e.part * heads;
  e.id = (size_t)e.bg * a.parts + e.part;
  e.len = min(max(a.length[e.bg / a.kv_heads], 0), a.capacity), e.m = min(e.len, a.keep);
  e.parts = (e.len + a.part_slots - 1) / a.part_slots;
  e.from = min(e.part * a.part_slots, e.len), e.to = min(e.len, e.from + a.part_slots);
  e.at = (int64_t)e.bg * a.capacity;
  return e;
}

__global__ __launch_bounds__(kSelThreads) void k_evict_keys(const EvictK a) {
  const EvictPart e = evict_part(a);
  const int tid = threadIdx.x, lane = tid & 63, b = e.bg / a.kv_heads;
  if (e.part == 0 && e.bg == b * a.kv_heads && tid == 0) a.length_out[b] = e.m;
  if (e.from >= e.to) return;
  constexpr int kRep = 4;  // exponents crowd
  __shared__ uint32_t hist[kBins1 * kRep];
  for (int x = tid; x < kBins1 * kRep; x += kSelThreads) hist[x] = 0;
  const int64_t recent_from = (int64_t)a.next_pos[b] - a.recent;
  __syncthreads();
  for (int j0 = e.from + tid; j0 < e.to; j0 += kPartSlots) {
    float f[kSelBatch];
    int p[kSelBatch];
#pragma unroll
    for (int t = 0; t < kSelBatch; ++t) {
      const int j = j0 + t * kSelThreads;
      f[t] = j < e.to ? ld_g(a.score + e.at + j) : 0.f;
      p[t] = j < e.to ? ld_g(a.pos + e.at + j) : 0;
    }
#pragma unroll
    for (int t = 0; t < kSelBatch; ++t) {
      const int j = j0 + t * kSelThreads;
      if (j >= e.to) continue;
      if (j < e.m) a.score_out[e.at + j] = f[t], a.pos_out[e.at + j] = p[t];  // k_evict_move overwrites the evicted ones
      if (e.m == e.len) continue;
      const uint32_t key = evict_key(p[t], f[t], recent_from, a.sinks);
      a.keys[e.at + j] = key;
      count_digit<kRep>(hist, key >> 22, lane);
    }
  }
  if (e.m == e.len) return;
  __syncthreads();
  uint32_t* out = a.hist + e.id * kBins1;
  for (int x = tid; x < kBins1; x += kSelThreads) {
    const uint4 c = reinterpret_cast<const uint4*>(hist)[x];
    out[x] = c.x + c.y + c.z + c.w;
  }
}

__global__ __launch_bounds__(kSelThreads) void k_evict_collect(const EvictK a) {
  constexpr int PER = kBins1 / kSelThreads;
  const EvictPart e = evict_part(a);
  if (e.m == e.len || e.from >= e.to) return;
  const int tid = threadIdx.x, lane = tid & 63;
  __shared__ uint32_t total_of[kSelWaves], picked[2], left, beyond;
  if (tid == 0) left = 0, beyond = 0;
  const uint32_t* hist = a.hist + (size_t)e.bg * a.parts * kBins1 + PER * tid;
  uint32_t c[PER] = {}, own[PER] = {};
#pragma unroll 8
  for (int p = 0; p < e.parts; ++p) {
    const uint2 x = *reinterpret_cast<const uint2*>(hist + (size_t)p * kBins1);
    c[0] += x.x, c[1] += x.y;
    if (p == e.part) own[0] = x.x, own[1] = x.y;
  }
  static_assert(PER == 2);
  pick_digit<kBins1>(c, e.m, total_of, picked);
  const uint32_t digit = picked[0];
  uint32_t above = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) above += (uint32_t)(PER * tid + j) > digit ? own[j] : 0u;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) above += __shfl_xor(above, o, 64);
  if (lane == 0 && above > 0) atomicAdd(&beyond, above);
  // The keys with that digit, in any order.
  for (int j0 = e.from + tid; j0 < e.to; j0 += kPartSlots) {
    uint32_t key[kSelBatch];
#pragma unroll
    for (int t = 0; t < kSelBatch; ++t) {
      const int j = j0 + t * kSelThreads;
      key[t] = j < e.to ? ld_g(a.keys + e.at + j) : 0u;
    }
#pragma unroll
    for (int t = 0; t < kSelBatch; ++t) {
      const bool in = j0 + t * kSelThreads < e.to && key[t] >> 22 == digit;
      const uint64_t who = __ballot(in);
      if (!in) continue;
      const int lead = __ffsll((unsigned long long)who) - 1;
      uint32_t first = 0;
      if (lane == lead) first = atomicAdd(&left, (uint32_t)__popcll(who));
      first = __shfl(first, lead, 64);
      a.few[e.at + e.from + first + __popcll(who & ((1ull << lane) - 1))] = key[t];
    }
  }
  __syncthreads();
  if (tid == 0) {
    a.part_of[e.id] = make_int2((int)left, (int)beyond);
    if (e.part == 0) a.digit[e.bg] = make_uint2(digit, picked[1]);
  }
}

__global__ __launch_bounds__(kSelThreads) void k_evict_lists(const EvictK a) {
  constexpr int W = kSelWaves, PER = kBins2 / kSelThreads;
  const EvictPart e = evict_part(a);
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (e.m == e.len) {
    if (e.part == 0 && tid == 0) a.count[e.bg] = 0;
    return;
  }
  if (e.from >= e.to) return;
  __shared__ uint32_t hist[kBins2];
  __shared__ uint32_t total_of[W], picked[2];
  __shared__ int tally[3][W];
  // What the first steps need is requested at once: the part's own keys, wave w's `run`
  // slots, 64 a turn; the head's digit; its parts' counts.
  const int run = ((e.to - e.from + 64 * W - 1) / (64 * W)) * 64, lo = min(e.to, e.from + wid * run);
  const int hi = min(e.to, lo + run);
  uint32_t own[kSelBatch];
#pragma unroll
  for (int t = 0; t < kSelBatch; ++t) {
    const int j = lo + t * 64 + lane;
    own[t] = j < hi ? ld_g(a.keys + e.at + j) : 0u;
  }
  const uint2 first = a.digit[e.bg];
  const int2 mine = lane < e.parts ? a.part_of[(size_t)e.bg * a.parts + lane] : make_int2(0, 0);
  // The keys of the head that share the digit: wave w has those of parts w, w + W, ..; the
  // first 64 kHold of a part stay in registers, f(key) sees each.
  constexpr int kHold = 10, kOwnParts = kMostParts / W;
  uint32_t held[kOwnParts][kHold];
  int held_n[kOwnParts];
#pragma unroll
  for (int z = 0; z < kOwnParts; ++z) {
    const int p = z * W + wid;
    held_n[z] = __builtin_amdgcn_readlane(mine.x, p);
    const uint32_t* few = a.few + e.at + (int64_t)p * a.part_slots + lane;
#pragma unroll
    for (int t = 0; t < kHold; ++t)
      if (t * 64 < held_n[z]) held[z][t] = t * 64 + lane < held_n[z] ? ld_g(few + t * 64) : 0u;
  }
  auto each_few = [&](int parts, auto&& f) {
#pragma unroll
    for (int z = 0; z < kOwnParts; ++z) {
      const int p = z * W + wid, n = held_n[z];
      if (p >= parts) continue;
#pragma unroll
      for (int t = 0; t < kHold; ++t)
        if (t * 64 + lane < n) f(held[z][t]);
      const uint32_t* few = a.few + e.at + (int64_t)p * a.part_slots;
      for (int x0 = kHold * 64 + lane; x0 < n; x0 += 64 * kSelBatch) {
        uint32_t key[kSelBatch];
#pragma unroll
        for (int t = 0; t < kSelBatch; ++t) key[t] = x0 + t * 64 < n ? ld_g(few + x0 + t * 64) : 0u;
#pragma unroll
        for (int t = 0; t < kSelBatch; ++t)
          if (x0 + t * 64 < n) f(key[t]);
      }
    }
  };
  uint32_t prefix = first.x, want = first.y;
#pragma unroll
  for (int shift = 11; shift >= 0; shift -= 11) {
    reinterpret_cast<uint4*>(hist)[tid] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    each_few(e.parts, [&](uint32_t key) {
      if (key >> (shift + 11) == prefix) count_digit<1>(hist, (key >> shift) & (kBins2 - 1), lane);
    });
    __syncthreads();
    static_assert(PER == 4);
    const uint4 x = reinterpret_cast<const uint4*>(hist)[tid];
    const uint32_t c[PER] = {x.x, x.y, x.z, x.w};
    pick_digit<kBins2>(c, want, total_of, picked);
    prefix = prefix << 11 | picked[0], want = picked[1];
    __syncthreads();  // before `picked` and `hist` are written again
  }
  // Kept: keys above prefix, and the first `want` slots with it.  Those of earlier parts:
  int above = 0, equal = 0;
  each_few(e.part, [&](uint32_t key) { above += key > prefix, equal += key == prefix; });
  if (wid == 0 && lane < e.part) above += mine.y;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) above += __shfl_xor(above, o, 64), equal += __shfl_xor(equal, o, 64);
  if (lane == 0) tally[0][wid] = above, tally[1][wid] = equal;
  __syncthreads();
  int kept = 0, ties = 0;
  for (int w = 0; w < W; ++w) kept += tally[0][w], ties += tally[1][w];
  __syncthreads();
  auto each = [&](auto&& f) {
    for (int j0 = lo; j0 < hi; j0 += 64 * kSelBatch) {
      uint32_t key[kSelBatch];
#pragma unroll
      for (int t = 0; t < kSelBatch; ++t) {
        const int j = j0 + t * 64 + lane;
        key[t] = j0 == lo ? own[t] : j < hi ? ld_g(a.keys + e.at + j) : 0u;
      }
#pragma unroll
      for (int t = 0; t < kSelBatch; ++t)
        if (j0 + t * 64 < hi) f(j0 + t * 64 + lane, key[t], j0 + t * 64 + lane < hi);
    }
  };
  above = 0, equal = 0;
  each([&](int, uint32_t key, bool in) {
    above += __popcll(__ballot(in && key > prefix)), equal += __popcll(__ballot(in && key == prefix));
  });
  if (lane == 0) tally[0][wid] = above, tally[1][wid] = equal;
  __syncthreads();
  for (int w = 0; w < wid; ++w) kept += tally[0][w], ties += tally[1][w];
  kept += min(ties, (int)want);
  // A slot below m that is evicted comes after (its slot - kept before) others; the kept
  // entries at or above m are listed from the last one down.
  const uint64_t below = (1ull << lane) - 1;
  int* hl = a.holes + (int64_t)e.bg * a.list;
  int* ml = a.movers + (int64_t)e.bg * a.list;
  each([&](int j, uint32_t key, bool in) {
    const uint64_t eq = __ballot(in && key == prefix);
    const bool k = in && (key > prefix || (key == prefix && ties + __popcll(eq & below) < (int)want));
    const uint64_t who = __ballot(k);
    const int before = kept + __popcll(who & below);
    if (in && j < e.m && !k) hl[j - before] = j;
    if (j >= e.m && k) ml[e.m - 1 - before] = j;
    if (in && j == e.m) a.count[e.bg] = e.m - before;
    ties += __popcll(eq), kept += __popcll(who);
  });
}

// Rows of the lists, `blocks` blocks a (sequence, head); with `entries`, their scores and
// positions too.
__global__ __launch_bounds__(256) void k_evict_move(const EvictK a, int blocks, bool entries) {
  const int bg = blockIdx.x / blocks, part = blockIdx.x - bg * blocks, b = bg / a.kv_heads, kvh = bg - b * a.kv_heads;
  const int pieces = a.row_bytes / 16;
  const int n = a.count[bg];
  const int64_t total = (int64_t)n * pieces, base = (b * a.c_row + kvh * a.c_head) * a.esz;
  const int64_t at = (int64_t)bg * a.capacity;
  const int* hl = a.holes + (int64_t)bg * a.list;
  const int* ml = a.movers + (int64_t)bg * a.list;
  for (int64_t x = part * 256 + threadIdx.x; x < total; x += (int64_t)blocks * 256) {
    const int r = (int)(x / pieces), piece = (int)(x - (int64_t)r * pieces), from = ml[n - 1 - r], to = hl[r];
    move_row(a, base, from, to, piece);
    if (entries && piece == 0) a.score_out[at + to] = a.score[at + from], a.pos_out[at + to] = a.pos[at + from];
  }
}

// Keys a lane in steps of 4, 256 slots: the threshold's search and the lists take a ballot a
// key.  1024 heads of 1200 slots with 20 / 24 / 32 keys 20.4 / 21.9 / 24.6 us.
template <int KPT>
void launch_short(const EvictK& a, int heads, hipStream_t s) {
  if constexpr (KPT * 64 < kShortSlots)
    if (a.capacity > KPT * 64) return launch_short<KPT + 4>(a, heads, s);
  hipLaunchKernelGGL(k_evict_short<KPT>, dim3(heads), dim3(256), 0, s, a);
}

// Most rows that a head can move; whether k_evict_short serves, and moves them itself.
int most_moves(const KvCache& c, int keep) { return std::max(0, std::min(keep, c.capacity - keep)); }
bool is_short(const KvCache& c) { return c.capacity <= kShortSlots; }
// Up to 16 KB of K rows a head: 1024 heads from 1056 to 1006, d 64, 18.7 us, with a kernel of
// its own for the moves 21.0; to 928 28.3 and 29.0; 32 heads to 928 12.7 and 14.5.
bool moves_within(const KvCache& c, int keep) {
  return is_short(c) && (size_t)most_moves(c, keep) * c.d * dtype_size(c.dt) <= 16 * 1024;
}
// Slots of a part of a long cache: the smallest that leave no more parts than the card
// takes at once, nor more than each block's sums over the parts' counts are worth: 8 heads of
// 131072 with 8 / 16 / 32 parts 83 / 67 / 60 us, 32 of 65536 with 8 / 17 169 / 166.
int part_slots(const KvCache& c) {
  const int heads = c.rows * c.kv_heads, parts = std::max(1, std::min(kMostParts, 1024 / std::max(1, heads)));
  const int64_t units = (c.capacity + (int64_t)kPartSlots - 1) / kPartSlots;
  return (int)((units + parts - 1) / parts * kPartSlots);
}
int parts_of(const KvCache& c) { return (int)((c.capacity + (int64_t)part_slots(c) - 1) / part_slots(c)); }

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
    // A step for each wave at least (2 x 16 heads of 2048, d 64: 5.4 us, with two 6.5, with
    // eight 13.3), and about eight blocks a CU (four to sixteen are the same).
    const int want = std::max(1, 2048 / std::max(1, c.rows * c.kv_heads));
    a.split_steps = std::max(kCommitWaves, (steps + want - 1) / want);
    a.splits = (steps + a.split_steps - 1) / a.split_steps;
  }
  // 4 x 8 heads of 16384, d 128: 32 rows 35.5 us with four tiles, 49 with one; 16 rows 34 and 32
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
  const size_t heads = (size_t)c.rows * c.kv_heads, parts = is_short(c) ? 0 : parts_of(c);
  const size_t of_long = is_short(c) ? 0 : 2 * (size_t)c.capacity + parts * (kBins1 + 2) + 2;
  return heads * (2 * (size_t)most_moves(c, keep) + 1 + of_long) * 4;
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
    uint32_t* at = static_cast<uint32_t*>(ws);
    auto take = [&](size_t n) { return std::exchange(at, at + n); };
    if (!is_short(c)) {
      a.parts = parts_of(c), a.part_slots = part_slots(c);
      a.hist = take((size_t)heads * a.parts * kBins1);
      a.part_of = reinterpret_cast<int2*>(take((size_t)heads * a.parts * 2));
      a.digit = reinterpret_cast<uint2*>(take((size_t)heads * 2));
      a.keys = take((size_t)heads * c.capacity);
      a.few = take((size_t)heads * c.capacity);
    }
    a.holes = reinterpret_cast<int*>(take((size_t)heads * a.list));
    a.movers = reinterpret_cast<int*>(take((size_t)heads * a.list));
    a.count = reinterpret_cast<int*>(take(heads));
  }
  if (is_short(c)) launch_short<4>(a, heads, s);
  else {
    const dim3 grid(heads * a.parts), block(kSelThreads);
    hipLaunchKernelGGL(k_evict_keys, grid, block, 0, s, a);
    hipLaunchKernelGGL(k_evict_collect, grid, block, 0, s, a);
    hipLaunchKernelGGL(k_evict_lists, grid, block, 0, s, a);
  }
  MRT_HIP_CHECK(hipGetLastError());
  if (a.holes != nullptr && a.list > 0) {
    const int64_t pieces = (int64_t)a.list * (a.row_bytes / 16);
    const int blocks = (int)std::max<int64_t>(1, std::min<int64_t>((pieces + 1023) / 1024, 8192 / heads));
    hipLaunchKernelGGL(k_evict_move, dim3(blocks * heads), dim3(256), 0, s, a, blocks, !is_short(c));
    MRT_HIP_CHECK(hipGetLastError());
  }
}

}  // namespace mrt
