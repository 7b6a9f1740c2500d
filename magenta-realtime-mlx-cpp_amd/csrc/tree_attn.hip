// Attention of a tree of drafted tokens over a cache.
//
// Node t of a sequence (parent -1: follows the cache; else an earlier node) attends
// every cache entry, its ancestors and itself:
//   s_tj = scale q_t . k_j + bias[h, min(distance, M - 1)],  out_t = softmax(s_t) V.
// One pass over the keys with the running maximum and sum of the softmax.
//
// Work: the n = heads / kv_heads query heads of a K/V head share its keys, so a K/V head
// (a unit) has R = nodes n rows r = t n + hq; its keys are taken in steps of 32, the
// drafted nodes the first ones.  Two kernels:
//   k_tree_few (up to 16 rows, fp32, odd head sizes): the four waves of a block take
//   steps in turn, straight from memory to registers, each with its own maximum, sum and
//   output; joined through LDS at the end.  What such rows cost is reading the keys.
//   k_tree_many (16-bit, d 64 or 128): eight waves, WR of them on different rows and
//   8 / WR on different steps, share K and V through a ring of LDS stages that loads
//   fill while products run.
// What they reach (bf16; one pass of the call, the joining of parts among it): 3 sequences
// of up to 65500 entries, 8 K/V heads, d 128, 60 rows (461 MB) 101 us, 4.6 TB/s, near the
// rate of a large copy; 16 of up to 8191, 4 K/V heads, 512 rows (79 GFLOP, half as much again
// for weights in two parts) 153 us, matrix cores busy for 33 % of the SIMDs' cycles and vector
// instructions (187 a wave and step against 48 matrix ones) for 42 %, which overlap little;
// fp32, 4 of up to 4099, 12 heads, 7 rows (58 MB) 25 us, bound by a few dependent trips to
// memory; one node over 49 entries 8 us of such trips.  Infinities among a cache's values cost
// a second round of steps (16 K/V heads of 4000 entries, 512 rows: 387 us instead of 58).
// A unit's steps are cut where the card needs more blocks (Share); parts leave (maximum,
// sum, output) in fp32 and k_tree_join sums them in order, so a result does not depend
// on timing.  The cut is made on the device, from the lengths, which the host never sees.
#include <algorithm>
#include <type_traits>

#include "attn_frag.hpp"
#include "kv_cache.hpp"
#include "mfma_ring.hpp"

namespace mrt {
namespace {

constexpr int kWaves = 4;
constexpr int kBiasLds = 4096;   // floats of the bias by distance kept in LDS

struct TreeArgs {
  const void *q, *k_new, *v_new, *k, *v;
  void* out;
  const int *parents, *length, *pos, *next_pos;
  const float* bias;
  float* lse;
  float* part;     // (slots, R, D) outputs of the parts
  float2* part_ml; // (slots, R) maximum (in log2 units) and sum
  uint64_t* present;  // (rows) mask of the nodes that are there
  int64_t q_row, q_node, q_head, kn_row, kn_node, kn_head, vn_row, vn_node, vn_head, o_row, o_node, o_head;
  int64_t c_row, c_head, c_slot, parents_stride;
  int rows, capacity, kv_heads, heads, nodes, D, buckets;
  int teams;       // parts of the whole work wanted, cut by all lengths; 0: each unit by itself,
  int splits;      //   into at most this many
  int least;       // steps that a part has at least
  int row_blocks;
  float scale;
};

__device__ __forceinline__ int steps_of(const TreeArgs& a, int b) {
  const int len = min(max(a.length[b], 0), a.capacity);
  return (len + kStepKeys - 1) / kStepKeys + (a.nodes + kStepKeys - 1) / kStepKeys;
}

// Work too small to be shared evenly: parts of a unit have max(least, ceil(steps /
// splits)) steps, part x of unit u leaves its result in slot u splits + x.  No block
// needs another sequence's length.
__device__ __forceinline__ int own_chunk(const TreeArgs& a, int steps) {
  return max(a.least, (steps + a.splits - 1) / a.splits);
}

// How the steps of all units (b, K/V head), in order, are cut into parts.  Long work
// (2 least, 16 steps, a team): each unit counts kUnitCost steps more, before its own, for beginning
// and ending it, and team t has the steps [t total / teams, (t + 1) total / teams), which
// may end and begin inside units; part t of unit u leaves its result in slot u + t.
// Short work: each unit is cut into parts of `chunk` steps, part t of all in slot t.
// Either way there are at most teams + units slots.
// Without that cost, 8 heads of 65500 entries beside 16 of 100 took 159 us (60 rows, d 128),
// the last team beginning and ending most of the short ones; with it 85.
constexpr int kUnitCost = 8;
struct Share {
  int64_t total;  // kUnitCost among it where chunk is 0
  int chunk;  // 0: by teams
};
// A value that all lanes hold, in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}
__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return uniform(v);
}
__device__ __forceinline__ Share share_of(const TreeArgs& a, int lane) {
  int64_t sum = 0;
  for (int b = lane; b < a.rows; b += 64) sum += steps_of(a, b);
  Share s;
  s.total = wave_sum64(sum) * a.kv_heads;
  s.chunk = s.total >= (int64_t)a.teams * a.least * 2 ? 0 : max(a.least, (int)((s.total + a.teams - 1) / a.teams));
  if (s.chunk == 0) s.total += (int64_t)kUnitCost * a.rows * a.kv_heads;
  return s;
}
// The sequence whose units hold position `at` of the running sum of count(b) kv_heads,
// and the sum before it; rows if there is none.
template <class Count>
__device__ __forceinline__ int find_row(const TreeArgs& a, int lane, int64_t at, int64_t* before, Count&& count) {
  int64_t base = 0;
  for (int b0 = 0; b0 < a.rows; b0 += 64) {
    int64_t incl = b0 + lane < a.rows ? (int64_t)count(b0 + lane) * a.kv_heads : 0;
    const int64_t own = incl;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t x = __shfl_up(incl, o, 64);
      if (lane >= o) incl += x;
    }
    const uint64_t past = __ballot(base + incl > at);
    if (past != 0) {
      const int l = __ffsll((unsigned long long)past) - 1;
      *before = uniform((int64_t)(base + __shfl(incl - own, l, 64)));
      return uniform(b0 + l);
    }
    base += uniform((int64_t)__shfl(incl, 63, 64));
  }
  return a.rows;
}
__device__ __forceinline__ int64_t team_of(const Share& s, int teams, int64_t at) {
  return ((at + 1) * teams + s.total - 1) / s.total - 1;
}

// Ancestor masks (own bit among them; 0: not there) of a sequence's nodes, by one wave:
// six doublings reach all 63 ancestors.
__device__ __forceinline__ uint64_t ancestors(const int* parents, int nodes, int lane) {
  int up = lane < nodes ? parents[lane] : -2;
  bool bad = up < -1 || up >= lane;
  if (bad) up = -1;
  uint64_t mask = 1ull << lane;
#pragma unroll
  for (int s = 0; s < 6; ++s) {
    const int from = up >= 0 ? up : lane;
    const uint32_t lo = __shfl((uint32_t)mask, from, 64), hi = __shfl((uint32_t)(mask >> 32), from, 64);
    const int up2 = __shfl(up, from, 64), bad2 = __shfl((int)bad, from, 64);
    if (up >= 0) {
      mask |= ((uint64_t)hi << 32) | lo;
      bad |= bad2 != 0;
      up = up2;
    }
  }
  return bad ? 0ull : mask;
}

// Whether a row's sum and outputs are numbers.
template <int E>
__device__ __forceinline__ bool all_finite(float l, const f32x4_t (&o)[E]) {
  float top = fabsf(l);
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int r = 0; r < 4; ++r) top = fmaf(0.f, o[e][r], top);  // NaN from either
  return top < INFINITY;
}

// E consecutive outputs of row r from dimension d on: to `out`, or, of a part, to its slot.
template <typename T, int E>
__device__ __forceinline__ void emit(const TreeArgs& a, bool whole, int64_t slot, int b, int kvh, int r, int d,
                                     const float (&v)[E], float top, float sum, bool there) {
  const int n = a.heads / a.kv_heads, node = r / n, h = kvh * n + r - node * n;
  if (whole) {
    there = there && sum != 0.f;
    const float inv = there ? 1.f / sum : 0.f;
    T* dst = static_cast<T*>(a.out) + b * a.o_row + node * a.o_node + h * a.o_head + d;
    union {
      T x[E];
      uint4 w4[(E * sizeof(T) + 15) / 16];
      uint2 w2;
      uint32_t w1;
    } u;
#pragma unroll
    for (int e = 0; e < E; ++e) u.x[e] = St<T>::st(there ? v[e] * inv : 0.f);
    if constexpr (E * sizeof(T) >= 16) {
#pragma unroll
      for (int w = 0; w < (int)(E * sizeof(T) / 16); ++w)
        if (d + w * (int)(16 / sizeof(T)) < a.D) reinterpret_cast<uint4*>(dst)[w] = u.w4[w];
    } else if (d < a.D) {
      if constexpr (E * sizeof(T) == 8) *reinterpret_cast<uint2*>(dst) = u.w2;
      else *reinterpret_cast<uint32_t*>(dst) = u.w1;
    }
    if (a.lse != nullptr && d == 0)
      a.lse[((size_t)b * a.nodes + node) * a.heads + h] = there ? fmaf(top, kLn2, logf(sum)) : -INFINITY;
  } else {
    const size_t at = slot * (size_t)(a.nodes * n) + r;
    float* dst = a.part + at * a.D + d;
    if constexpr (E % 4 == 0) {
#pragma unroll
      for (int e = 0; e < E; e += 4)
        if (d + e < a.D) *reinterpret_cast<float4*>(dst + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    } else if (d < a.D) {
      *reinterpret_cast<float2*>(dst) = make_float2(v[0], v[1]);
    }
    if (d == 0) a.part_ml[at] = make_float2(top, sum);
  }
}

// Blocks of k_tree_few that a CU holds at least: its registers without the rare second
// round of steps would let it hold as many.
constexpr int few_blocks(size_t elt, int dp, int nr) {
  return elt == 4 ? 1 : dp == 32 ? (nr == 1 ? 4 : nr == 2 ? 3 : 2) : dp * nr <= 128 ? 2 : 1;
}

template <typename T, int DP, int NR>
__global__ __launch_bounds__(64 * kWaves, few_blocks(sizeof(T), DP, NR)) void k_tree_few(const TreeArgs a) {
  using F = AttnFrag<T, DP>;
  constexpr int E = F::E, VW = F::VW, KC = F::KC;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4, D = a.D;
  const int id = blockIdx.x / a.row_blocks, row0 = (blockIdx.x - id * a.row_blocks) * (16 * NR);
  const int new_steps = (a.nodes + kStepKeys - 1) / kStepKeys;
  int b, kvh, s0, s1, steps;
  if (a.teams == 0) {
    const int unit = id / a.splits;
    b = unit / a.kv_heads, kvh = unit - b * a.kv_heads;
    s0 = 0;
  } else {
    const Share sh = share_of(a, lane);
    const int chunk = sh.chunk > 0 ? sh.chunk : (int)((sh.total + a.teams - 1) / a.teams);
    auto parts = [&](int x) { return (steps_of(a, x) + chunk - 1) / chunk; };
    int64_t before = 0;
    b = find_row(a, lane, id, &before, parts);
    if (b >= a.rows) return;
    const int n = parts(b), at = (int)(id - before);
    kvh = at / n;
    steps = steps_of(a, b);
    s0 = (at - kvh * n) * chunk, s1 = min(steps, s0 + chunk);
  }
  if (a.teams == 0 && a.splits > 1) {
    const int part = id - (b * a.kv_heads + kvh) * a.splits;
    steps = steps_of(a, b);
    const int chunk = own_chunk(a, steps);
    s0 = part * chunk, s1 = min(steps, s0 + chunk);
    if (s0 >= steps) return;
  }
  const int n = a.heads / a.kv_heads, R = a.nodes * n;
  const T* kc = static_cast<const T*>(a.k) + b * a.c_row + kvh * a.c_head;
  const T* vc = static_cast<const T*>(a.v) + b * a.c_row + kvh * a.c_head;
  const int* pos = a.pos == nullptr ? nullptr : a.pos + (size_t)(b * a.kv_heads + kvh) * a.capacity;

  // Keys, values and positions of a step.  Nothing here needs the length (rows past it are masked,
  // those past the capacity are read from its last slot), so a wave's first step is
  // requested before anything else.
  uint4 kf[2][KC];
  uint32_t vf[8][VW];
  int kpos[8];
  auto load = [&](int st) {
    const bool fresh = st < new_steps;  // drafted nodes
    const int base = (fresh ? st : st - new_steps) * kStepKeys, last = (fresh ? a.nodes : a.capacity) - 1;
    const T* kb = fresh ? static_cast<const T*>(a.k_new) + b * a.kn_row + kvh * a.kn_head : kc;
    const T* vb = fresh ? static_cast<const T*>(a.v_new) + b * a.vn_row + kvh * a.vn_head : vc;
    const int64_t kstep = fresh ? a.kn_node : a.c_slot, vstep = fresh ? a.vn_node : a.c_slot;
#pragma unroll
    for (int h = 0; h < 2; ++h) F::load_row(kb + (int64_t)min(base + step_key(i, h), last) * kstep, g, D, kf[h]);
#pragma unroll
    for (int j = 0; j < 8; ++j) F::load_v(vb + (int64_t)min(base + lane_key(g, j), last) * vstep, i, D, vf[j]);
    if (a.bias != nullptr && pos != nullptr && !fresh) {
#pragma unroll
      for (int j = 0; j < 8; ++j) kpos[j] = ld_g(pos + min(base + lane_key(g, j), last));
    }
  };
  load(s0 + wid);
  // Of cached step `st` or the nodes', element j of V once more.
  auto load_v = [&](bool fresh, int key, uint32_t (&f)[VW]) {
    F::load_v(fresh ? static_cast<const T*>(a.v_new) + b * a.vn_row + kvh * a.vn_head + (int64_t)key * a.vn_node
                    : vc + (int64_t)key * a.c_slot,
              i, D, f);
  };

  const int len = min(max(a.length[b], 0), a.capacity), old_steps = (len + kStepKeys - 1) / kStepKeys;
  if (a.teams == 0 && a.splits == 1) s1 = steps = new_steps + old_steps;
  const bool all = s0 == 0 && s1 == steps;

  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ uint64_t sees[kMaxNodes];
  __shared__ float2 ml[kWaves][16 * NR];
  float* btab = reinterpret_cast<float*>(lds);  // the bias of this K/V head's heads, until the waves join
  const bool bias_in_lds = n * a.buckets <= kBiasLds;

  uint4 q[NR][KC];
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    const int r = min(row0 + t * 16 + i, R - 1), node = r / n;
    F::load_row(static_cast<const T*>(a.q) + b * a.q_row + node * a.q_node + (int64_t)(kvh * n + r - node * n) * a.q_head,
                g, D, q[t]);
  }
  if (wid == 0) sees[lane] = ancestors(a.parents + b * a.parents_stride, a.nodes, lane);
  if (a.bias != nullptr && bias_in_lds)
    for (int x = tid; x < n * a.buckets; x += 64 * kWaves) btab[x] = a.bias[(size_t)kvh * n * a.buckets + x];
  ring_barrier();  // does not wait for the loads of the first step

  int qpos[NR];
  const float* brow[NR];
  if (a.bias != nullptr) {
    const int first = a.next_pos != nullptr ? a.next_pos[b] : len;
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      const int r = min(row0 + t * 16 + i, R - 1), node = r / n, hq = r - node * n;
      qpos[t] = first + max(__popcll(sees[node]) - 1, 0);
      brow[t] = (bias_in_lds ? btab : a.bias + (size_t)kvh * n * a.buckets) + hq * a.buckets;
    }
  }

  f32x4_t o[NR][E];
  float m[NR], l[NR];
  auto begin = [&] {
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      m[t] = kNone, l[t] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[t][e] = {0.f, 0.f, 0.f, 0.f};
    }
  };
  begin();
  const float scale2 = a.scale * kLog2e;
  // fp16 weights reach up to 2^15, so that those far below the maximum keep their bits.
  constexpr float kShift = std::is_same_v<T, f16> ? 15.f : 0.f;

  // One step.  A matrix product makes NaN of 0 * inf, and of infinities whose weight is in
  // two parts: a node's infinities and NaN, which others may not see, are left out of it and
  // added by class; with `exact`, the cache's are too, and masked entries' keys have no part.
  auto step = [&](int st, auto exact) {
    const bool fresh = st < new_steps;
    const int base = (fresh ? st : st - new_steps) * kStepKeys, end = fresh ? a.nodes : len;
    const bool whole = base + kStepKeys <= end;
    if (!whole) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int w = 0; w < VW; ++w) vf[j][w] = base + lane_key(g, j) < end ? vf[j][w] : 0u;
    }
    float p[NR][8];
    if (a.bias != nullptr && (fresh || pos == nullptr)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = min(base + lane_key(g, j), end - 1);
        kpos[j] = fresh ? __popcll(sees[key]) - 1 : key;
      }
    }
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      const f32x4_t x = F::scores(kf[0], q[t]), y = F::scores(kf[1], q[t]);
      const float s[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      const int node = min(row0 + t * 16 + i, R - 1) / n;
      if (a.bias != nullptr) {
        const int at = fresh ? __popcll(sees[node]) - 1 : qpos[t];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float by = brow[t][bucket(at, kpos[j], a.buckets)] * kLog2e;
          p[t][j] = fmaf(s[j], scale2, by);
          if (exact.value && by < kNone) p[t][j] = -INFINITY;  // masked, whatever the key holds
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[t][j] = s[j] * scale2;
      }
      if (fresh) {
        const uint64_t see = sees[node] >> base;
#pragma unroll
        for (int j = 0; j < 8; ++j) p[t][j] = (see >> lane_key(g, j)) & 1 ? p[t][j] : -INFINITY;
      } else if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[t][j] = base + lane_key(g, j) < end ? p[t][j] : -INFINITY;
      }
    }
    uint32_t seen[NR];  // the keys that the row does not mask, a bit each
    if (fresh || exact.value) {
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        seen[t] = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) seen[t] |= p[t][j] < kNone ? 0u : 1u << j;
      }
    }
    running_softmax<NR, E>(p, m, l, o, kShift);
    if (!fresh && !exact.value) {
      F::template add_pv<NR>(vf, p, o);
    } else {
      uint32_t diff = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          const uint32_t x = F::finite_part(vf[j][w]);
          diff |= x ^ vf[j][w];
          vf[j][w] = x;
        }
      F::template add_pv<NR>(vf, p, o);
      if (__builtin_expect(__any(diff != 0), 0)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = base + lane_key(g, j);
          load_v(fresh, min(key, end - 1), vf[j]);
#pragma unroll
          for (int w = 0; w < VW; ++w) vf[j][w] = key < end ? F::classes(vf[j][w]) : 0u;
        }
#pragma unroll
        for (int t = 0; t < NR; ++t) {
          float one[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) one[j] = (seen[t] >> j) & 1 ? 1.f : 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const f32x4_t c = F::count(vf, one, e);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[t][e][r] += F::class_value(c[r]);
          }
        }
      }
    }
  };
  for (int st = s0 + wid; st < s1; st += kWaves) {
    step(st, std::false_type{});
    if (st + kWaves < s1) load(st + kWaves);
  }
  bool odd = false;
#pragma unroll
  for (int t = 0; t < NR; ++t) odd |= !all_finite<E>(l[t], o[t]) && sees[min(row0 + t * 16 + i, R - 1) / n] != 0;
  if (__builtin_expect(__any(odd), 0)) {  // rare: this wave's steps once more
    begin();
#pragma unroll 1
    for (int st = s0 + wid; st < s1; st += kWaves) {
      load(st);
      step(st, std::true_type{});
    }
  }

  // Join the waves: outputs at the common maximum, summed through LDS.
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    l[t] = sum_over_groups(l[t]);
    if (g == 0) ml[wid][t * 16 + i] = make_float2(m[t], l[t]);
  }
  __syncthreads();  // and the bias in LDS has been read
  f32x4_t* buf = reinterpret_cast<f32x4_t*>(lds);
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    float top = ml[0][t * 16 + i].x;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, ml[w][t * 16 + i].x);
    const float f = fade(m[t] - top);
#pragma unroll
    for (int e = 0; e < E; ++e) buf[((wid * NR + t) * E + e) * 64 + lane] = o[t][e] * f;
  }
  __syncthreads();
  // Thread (lane, r = wid): dimensions (4 g + r) E .. + E - 1 of row i of each tile.
  const int64_t slot = id;
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    const int r = row0 + t * 16 + i, d = (4 * g + wid) * E;
    if (r >= R) continue;
    float top = ml[0][t * 16 + i].x, sum = 0.f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, ml[w][t * 16 + i].x);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum = fmaf(ml[w][t * 16 + i].y, __builtin_amdgcn_exp2f(ml[w][t * 16 + i].x - top), sum);
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) v[e] += reinterpret_cast<const float*>(&buf[((w * NR + t) * E + e) * 64 + lane])[wid];
    }
    emit<T, E>(a, all, slot, b, kvh, r, d, v, top, sum, sees[r / n] != 0);
  }
  if (!all && s0 == 0 && row0 == 0 && wid == 0) {  // the same from every K/V head
    const uint64_t there = __ballot(sees[lane] != 0);
    if (lane == 0) a.present[b] = there;
  }
}

// ---- many rows ---------------------------------------------------------------------

template <int DP, int WR, int NR>
struct Many {
  static constexpr int kWaves = 8, WK = kWaves / WR, kKeys = 32 * WK;  // keys of a stage
  static constexpr int kRow = 2 * DP, kStage = 2 * kKeys * kRow;       // bytes: a key, K and V of a stage
  static constexpr bool kHalves = WR == 8;                             // two halves of the waves, half a step apart
  static constexpr int S = kStage >= 64 * 1024 ? 2 : kHalves ? 5 : 4;  // stages
  static constexpr int kLoads = kStage / 1024 / kWaves;  // 1 KB loads of a wave and stage
  static constexpr int kPieces = kRow / 16, kRowsLoad = 1024 / kRow;
  static constexpr size_t kRing = (size_t)S * kStage, kJoin = WK > 1 ? (size_t)kWaves * NR * (DP / 16) * 1024 : 0;
  static constexpr size_t kLds = kRing > kJoin ? kRing : kJoin;
  // 16-byte piece p of row r lies at place p ^ swz(r), so that what is read together falls
  // in distinct banks: of K the same piece of 16 keys, of V 32 bytes of 8 keys.
  __device__ static int swz_k(int r) { return DP == 128 ? r & 15 : (r >> 1) & 7; }
  __device__ static int swz_v(int r) { return DP == 128 ? (r & 7) * 2 : ((r >> 1) & 3) * 2; }
};

// 1 KB of a stage: lane l's 16 bytes from `base` + `off` (or `from`) to LDS address `to` +
// 16 l.  Written out, since before any read of LDS the compiler waits for every such load
// that it knows of, which would empty the ring; the waits below count them.  No register
// is written; m0, which nothing else here uses, is set in the same place.  What the
// compiler counts itself only gets longer by these loads.
__device__ __forceinline__ void load_lds(uint32_t to, const void* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void load_lds(uint32_t to, const void* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}
// V, transposed as it is read: of 16 lanes, lane 4 r + c gives the address of columns 4 c ..
// 4 c + 3 of row r, and lane i receives column i of rows 0..3.
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u32x2_t read_transposed(uint32_t at) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((MRT_LDS s4*)(uintptr_t)at));
}
__device__ __forceinline__ uint4 read_lds16(uint32_t at) {
  return __builtin_bit_cast(uint4, *(const MRT_LDS u32x4_t*)(uintptr_t)at);
}

template <typename T, int DP, int WR, int NR, bool BIAS>
__global__ __launch_bounds__(512) void k_tree_many(const TreeArgs a) {
  using F = AttnFrag<T, DP>;
  using M = Many<DP, WR, NR>;
  constexpr int E = F::E, KC = F::KC, WK = M::WK, S = M::S;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4, wr = wid % WR, wk = wid / WR;
  // The row blocks of a team share keys: they follow each other on one XCD.
  const int id = blockIdx.x >> 3, rb = id % a.row_blocks;
  const int64_t team = (int64_t)(id / a.row_blocks) * 8 + (blockIdx.x & 7);
  const int n = a.heads / a.kv_heads, R = a.nodes * n, row0 = (rb * WR + wr) * (16 * NR);
  // Logits in log2 units are mult z: z the products themselves, whose sign q takes on, or
  // with a bias the finished logits.  Not 0, which would make NaN of a masked -inf.
  const float size = fabsf(a.scale) * kLog2e, scale2 = size < 1e-37f ? 1e-37f : size, mult = BIAS ? 1.f : scale2;
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
  // The maximum that the weights refer to follows only where a logit passes it by more
  // than kSlack: most steps then leave the output alone.  fp16 weights stay below 2^15.
  constexpr float kSlack = 8.f, kShift = std::is_same_v<T, f16> ? 15.f - kSlack : 0.f;

  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ uint64_t sees[kMaxNodes];
  __shared__ float2 ml[WK][16 * NR * WR];
  float* btab = reinterpret_cast<float*>(lds + M::kLds);
  const uint32_t ring = (uint32_t)(uintptr_t)(MRT_LDS char*)lds;  // LDS address of the ring
  uint32_t k_at[KC], v_at[E];  // in a stage: this lane's key row and chunk; V row and columns
#pragma unroll
  for (int c = 0; c < KC; ++c) k_at[c] = (wk * 32 + i) * M::kRow + ((c * 4 + g) ^ M::swz_k(i)) * 16;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int row = 4 * g + (i >> 2), piece = 2 * e + ((i >> 1) & 1);
    v_at[e] = (M::kKeys + wk * 32 + row) * M::kRow + (piece ^ M::swz_v(row)) * 16 + (i & 1) * 8;
  }
  // Where this lane's part of each load lies behind a stage's first key (whole stages).
  uint32_t src[M::kLoads];
  const bool near = a.c_slot < (1 << 23);
#pragma unroll
  for (int x = 0; x < M::kLoads; ++x) {
    const int t = x * M::kWaves + wid, half = M::kLoads * M::kWaves / 2, u = t < half ? t : t - half;
    const int row = u * M::kRowsLoad + lane / M::kPieces, place = lane % M::kPieces;
    src[x] = ((uint32_t)row * (uint32_t)a.c_slot + (place ^ (t < half ? M::swz_k(row & 31) : M::swz_v(row))) * 8) * 2;
  }
  const bool bias_in_lds = n * a.buckets <= kBiasLds;

  // This block's part of the work: steps [at, stop) of the running order, from unit
  // (b, kvh) whose first step is at `unit_at`.
  int b, kvh;
  int64_t at, stop, unit_at;
  Share sh{0, 0};
  if (a.teams == 0) {
    const int unit = (int)team / a.splits, part = (int)team - unit * a.splits;
    if (unit >= a.rows * a.kv_heads) return;
    b = unit / a.kv_heads, kvh = unit - b * a.kv_heads;
    const int steps = steps_of(a, b), chunk = a.splits > 1 ? own_chunk(a, steps) : steps;
    unit_at = 0, at = (int64_t)part * chunk, stop = min((int64_t)steps, at + chunk);
  } else {
    sh = share_of(a, lane);
    int64_t before = 0;
    if (sh.chunk > 0) {
      auto parts = [&](int x) { return (steps_of(a, x) + sh.chunk - 1) / sh.chunk; };
      b = find_row(a, lane, team, &before, parts);
      if (b >= a.rows) return;
      const int np = parts(b), x = (int)(team - before);
      kvh = x / np;
      unit_at = 0, at = (int64_t)(x - kvh * np) * sh.chunk, stop = min((int64_t)steps_of(a, b), at + sh.chunk);
    } else {
      if (team >= a.teams) return;
      at = team * sh.total / a.teams, stop = (team + 1) * sh.total / a.teams;
      b = find_row(a, lane, at, &before, [&](int x) { return kUnitCost + steps_of(a, x); });
      const int per = kUnitCost + steps_of(a, b);
      kvh = (int)((at - before) / per);
      unit_at = before + (int64_t)kvh * per + kUnitCost;
    }
  }
  b = uniform(b), kvh = uniform(kvh), at = uniform(at), stop = uniform(stop), unit_at = uniform(unit_at);

  while (at < stop) {
    const int len = uniform(min(max(a.length[b], 0), a.capacity)), old_steps = (len + kStepKeys - 1) / kStepKeys;
    const int new_steps = (a.nodes + kStepKeys - 1) / kStepKeys, steps = new_steps + old_steps;
    const int s0 = (int)max(at - unit_at, (int64_t)0), s1 = (int)min((int64_t)steps, stop - unit_at);
    if (s1 <= 0) break;  // the next team begins this unit
    const bool all = s0 == 0 && s1 == steps;
    const T* kc = static_cast<const T*>(a.k) + b * a.c_row + kvh * a.c_head;
    const T* vc = static_cast<const T*>(a.v) + b * a.c_row + kvh * a.c_head;
    const int stages = (s1 - s0 + WK - 1) / WK;

    // Requests the next stage (past the end: the last step again): K rows, then V rows.
    const int64_t stride = (int64_t)M::kKeys * a.c_slot * 2;  // bytes of a stage's keys
    const char* kb = reinterpret_cast<const char*>(kc + (int64_t)(s0 - new_steps) * kStepKeys * a.c_slot);
    const char* vb = reinterpret_cast<const char*>(vc + (int64_t)(s0 - new_steps) * kStepKeys * a.c_slot);
    int ahead = s0, to_slot = 0;
    const int plain_to = near ? min(s1, new_steps + len / kStepKeys) : 0;  // whole cached steps end here
    auto issue = [&] {
      const uint32_t to = ring + to_slot * M::kStage;
      to_slot = to_slot + 1 == S ? 0 : to_slot + 1;
      const int first = ahead;
      ahead += WK;
      if (first >= new_steps && ahead <= plain_to) {
#pragma unroll
        for (int x = 0; x < M::kLoads; ++x) {
          const int t = x * M::kWaves + wid;
          load_lds(to + t * 1024, x < M::kLoads / 2 || (M::kLoads == 1 && wid < M::kWaves / 2) ? kb : vb, src[x]);
        }
      } else {
        const T* kn = static_cast<const T*>(a.k_new) + b * a.kn_row + kvh * a.kn_head;
        const T* vn = static_cast<const T*>(a.v_new) + b * a.vn_row + kvh * a.vn_head;
#pragma unroll
        for (int x = 0; x < M::kLoads; ++x) {
          const int t = x * M::kWaves + wid, half = M::kLoads * M::kWaves / 2, u = t < half ? t : t - half;
          const int row = u * M::kRowsLoad + lane / M::kPieces, place = lane % M::kPieces;
          const int st = min(first + u * M::kRowsLoad / 32, s1 - 1);
          const bool fresh = st < new_steps;
          const int key = min((fresh ? st : st - new_steps) * kStepKeys + (row & 31), (fresh ? a.nodes : len) - 1);
          const T* from = t < half ? (fresh ? kn + key * a.kn_node : kc + key * a.c_slot) + (place ^ M::swz_k(row & 31)) * 8
                                   : (fresh ? vn + key * a.vn_node : vc + key * a.c_slot) + (place ^ M::swz_v(row)) * 8;
          load_lds(to + t * 1024, from);
        }
      }
      kb += stride, vb += stride;
    };
    uint4 q[NR][KC];
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      const int r = min(row0 + t * 16 + i, R - 1), node = r / n;
      F::load_row(static_cast<const T*>(a.q) + b * a.q_row + node * a.q_node + (int64_t)(kvh * n + r - node * n) * a.q_head,
                  g, DP, q[t]);
    }
#pragma unroll
    for (int t = 0; t < NR; ++t)
#pragma unroll
      for (int c = 0; c < KC; ++c) q[t][c].x ^= flip, q[t][c].y ^= flip, q[t][c].z ^= flip, q[t][c].w ^= flip;
    if (wid == 0) sees[lane] = ancestors(a.parents + b * a.parents_stride, a.nodes, lane);
    if (BIAS && bias_in_lds)
      for (int x = tid; x < n * a.buckets; x += 512) btab[x] = a.bias[(size_t)kvh * n * a.buckets + x];
    const int first_pos = BIAS && a.next_pos != nullptr ? a.next_pos[b] : len;
    // From here on the only vector memory operations are the stages' (but for a bias
    // with positions or too large for LDS, whose loads make waits longer, not shorter).
#pragma unroll
    for (int s = 0; s < (M::kHalves ? S - 2 : S - 1); ++s) issue();

    f32x4_t o[NR][E];  // [t][e][r]: dimension 16 e + 4 g + r of row i of tile t
    float m[NR], l[NR];
    auto begin = [&] {
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        m[t] = kNone, l[t] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[t][e] = {0.f, 0.f, 0.f, 0.f};
      }
    };
    begin();

    // A step: where its keys are, whether they are nodes, and whether all 32 count for all.
    struct Step {
      uint32_t stage;
      int base, end;
      bool on, fresh, plain;
    };
    int slot_now = 0;
    auto step_of = [&](int s) {
      Step p;
      p.stage = ring + slot_now * M::kStage;
      slot_now = slot_now + 1 == S ? 0 : slot_now + 1;
      const int st = s0 + s * WK + wk;
      p.on = st < s1 && row0 < R;
      p.fresh = st < new_steps;
      p.base = (p.fresh ? st : st - new_steps) * kStepKeys, p.end = p.fresh ? a.nodes : len;
      p.plain = !p.fresh && p.base + kStepKeys <= len;
      return p;
    };
    f32x4_t x[NR], y[NR];  // Q K^T of a step
    uint4 ph[NR], pl[NR];  // its weights
    uint32_t seen[NR];     // with `exact`: the keys that the row does not mask, a bit each
    uint32_t left_out = 0;  // nonzero: infinities or NaN among the nodes' values
    auto scores = [&](const Step& p) {
      const uint32_t stage = p.stage;
#pragma unroll
      for (int t = 0; t < NR; ++t) x[t] = {0.f, 0.f, 0.f, 0.f}, y[t] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c0 = 0; c0 < KC; c0 += 2) {
        uint4 kx[2][2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          kx[0][c] = read_lds16(stage + k_at[c0 + c]);
          kx[1][c] = read_lds16(stage + k_at[c0 + c] + 16 * M::kRow);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int t = 0; t < NR; ++t) {
            x[t] = Mma<T>::mma(kx[0][c], q[t][c0 + c], x[t]);
            y[t] = Mma<T>::mma(kx[1][c], q[t][c0 + c], y[t]);
          }
      }
    };
    auto weights = [&](const Step& w, auto only) {  // of all row tiles, or with `exact` of one
      constexpr bool exact = only.value >= 0;
      constexpr int t0 = exact ? only.value : 0, t1 = exact ? t0 + 1 : NR;
      const bool fresh = w.fresh, plain = w.plain;
      const int base = w.base, end = w.end;
      float z[NR][8];
#pragma unroll
      for (int t = t0; t < t1; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) z[t][j] = x[t][j], z[t][4 + j] = y[t][j];
      if constexpr (BIAS) {
        const int* pos = a.pos == nullptr ? nullptr : a.pos + (size_t)(b * a.kv_heads + kvh) * a.capacity;
        int kpos[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = min(base + lane_key(g, j), end - 1);
          kpos[j] = fresh ? __popcll(sees[key]) - 1 : pos != nullptr ? pos[key] : key;
        }
#pragma unroll
        for (int t = t0; t < t1; ++t) {
          const int r = min(row0 + t * 16 + i, R - 1), node = r / n, hq = r - node * n;
          const int qp = (fresh ? 0 : first_pos) + max(__popcll(sees[node]) - 1, 0);
          const float* row = (bias_in_lds ? btab : a.bias + (size_t)kvh * n * a.buckets) + hq * a.buckets;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float by = row[bucket(qp, kpos[j], a.buckets)] * kLog2e;
            z[t][j] = fmaf(z[t][j], scale2, by);
            if (exact && by < kNone) z[t][j] = -INFINITY;  // masked, whatever the key holds
          }
        }
      }
      if (!plain) {
#pragma unroll
        for (int t = t0; t < t1; ++t) {
          const uint64_t see = fresh ? sees[min(row0 + t * 16 + i, R - 1) / n] >> base : ~0ull;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            z[t][j] = base + lane_key(g, j) < end && (see >> lane_key(g, j)) & 1 ? z[t][j] : -INFINITY;
        }
      }
      if constexpr (exact) {
#pragma unroll
        for (int t = t0; t < t1; ++t) {
          seen[t] = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) seen[t] |= z[t][j] * mult < kNone ? 0u : 1u << j;
        }
      }
#pragma unroll
      for (int t = t0; t < t1; ++t) {
        const float top = max_over_groups(fmaxf(fmaxf(fmaxf(z[t][0], z[t][1]), fmaxf(z[t][2], z[t][3])),
                                                fmaxf(fmaxf(z[t][4], z[t][5]), fmaxf(z[t][6], z[t][7])))) *
                              mult -
                          kShift;
        if (__any(top > m[t] + kSlack)) {  // each row by itself: its bits do not depend on the others'
          const float mn = top > m[t] + kSlack ? top : m[t], f = fade(m[t] - mn);
          m[t] = mn;
          l[t] *= f;
#pragma unroll
          for (int e = 0; e < E; ++e) o[t][e] *= f;
        }
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(z[t][j], mult, -m[t]));
        l[t] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        F::split(p, ph[t], pl[t]);
      }
    };
    auto values = [&](const Step& p) {
      const uint32_t stage = p.stage;
      const bool fresh = p.fresh, plain = p.plain;
      const int base = p.base, end = p.end;
      // Rows past the end are zeros; a node's infinities and NaN belong to those who see it
      // and are added in the end.
#pragma unroll
      for (int e0 = 0; e0 < E; e0 += 4) {
        u32x2_t vx[4][2];  // keys 16 h + 4 g .. + 3 of dimension 16 e + i
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          vx[e][0] = read_transposed(stage + v_at[e0 + e]);
          vx[e][1] = read_transposed(stage + v_at[e0 + e] + 16 * M::kRow);
        }
        if (!plain) {
          uint32_t in[2][2];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const int key = base + 16 * h + 4 * g + 2 * w;
              in[h][w] = (key < end ? 0xffffu : 0u) | (key + 1 < end ? 0xffff0000u : 0u);
            }
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int w = 0; w < 2; ++w) {
                const uint32_t v = vx[e][h][w] & in[h][w], u = fresh ? F::finite_part(v) : v;
                left_out |= u ^ v;
                vx[e][h][w] = u;
              }
        }
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int t = 0; t < NR; ++t)
              o[t][e0 + e] = Mma<T>::mma(make_uint4(vx[e][0].x, vx[e][0].y, vx[e][1].x, vx[e][1].y), part == 0 ? ph[t] : pl[t],
                                         o[t][e0 + e]);
      }
    };

    if constexpr (M::kHalves) {
      // Two halves of the block, a wave of each on every SIMD, half a step apart: while one
      // multiplies (Q K^T of step s, P V of step s - 1), the other has its softmax.  Every
      // wave passes 2 stages + 1 barriers; barrier 2 s comes after everyone's loads of
      // stage s and the last read of stage s - 2.
      constexpr int kWait = (S - 3) * M::kLoads;
      const bool second = wid >= M::kWaves / 2;
      if (second) {
        __builtin_amdgcn_s_waitcnt(vm_wait_imm(kWait));
        ring_barrier();
        issue();
      }
      Step prev{};  // each stage is a step here; waves without rows compute along and write nothing
      for (int s = 0; s < stages; ++s) {
        if (!second) __builtin_amdgcn_s_waitcnt(vm_wait_imm(kWait));
        ring_barrier();
        if (!second) issue();
        const Step now = step_of(s);
        scores(now);
        if (s > 0) values(prev);
        if (second) __builtin_amdgcn_s_waitcnt(vm_wait_imm(kWait));
        ring_barrier();
        if (second) issue();
        weights(now, std::integral_constant<int, -1>{});
        prev = now;
      }
      if (!second) ring_barrier();
      values(prev);
    } else {
      for (int s = 0; s < stages; ++s) {
        __builtin_amdgcn_s_waitcnt(vm_wait_imm((S - 2) * M::kLoads));  // this wave's part of stage s is in LDS
        ring_barrier();                                                // everyone's is, and stage s - 1 has been read
        issue();
        const Step now = step_of(s);
        if (!now.on) continue;
        scores(now);
        weights(now, std::integral_constant<int, -1>{});
        values(now);
      }
    }

    if (__builtin_expect(__any(left_out != 0), 0)) {  // rare, so from memory; by class as above
      const uint16_t* vn = static_cast<const uint16_t*>(a.v_new) + b * a.vn_row + kvh * a.vn_head;
      for (int st = s0 + wk; st < min(s1, new_steps); st += WK) {
        const int base = st * kStepKeys;
#pragma unroll
        for (int t = 0; t < NR; ++t) {
          const uint64_t see = sees[min(row0 + t * 16 + i, R - 1) / n] >> base;
          uint32_t one[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            one[j] = Mma<T>::pack((see >> lane_key(g, 2 * j)) & 1 ? 1.f : 0.f, (see >> lane_key(g, 2 * j + 1)) & 1 ? 1.f : 0.f);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            uint32_t c[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int key = base + 16 * (w >> 1) + 4 * g + 2 * (w & 1), last = a.nodes - 1;
              c[w] = F::classes(ld_g(vn + min(key, last) * a.vn_node + 16 * e + i) |
                                (uint32_t)ld_g(vn + min(key + 1, last) * a.vn_node + 16 * e + i) << 16);
            }
            const f32x4_t sum = Mma<T>::mma(make_uint4(c[0], c[1], c[2], c[3]), make_uint4(one[0], one[1], one[2], one[3]),
                                            f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int r = 0; r < 4; ++r) o[t][e][r] += F::class_value(sum[r]);
          }
        }
      }
    }
    // Where something did not stay finite (see k_tree_few), the wave takes its steps once
    // more, from memory, with all infinities and NaN of V added by class.
    bool odd = false;
#pragma unroll
    for (int t = 0; t < NR; ++t) odd |= !all_finite<E>(l[t], o[t]) && sees[min(row0 + t * 16 + i, R - 1) / n] != 0;
    if (__builtin_expect(row0 < R && __any(odd), 0)) {
      begin();
      // One row tile after the other, no loads ahead: what this takes in registers, the loops
      // above would have to do without.
      auto tile = [&](auto only) {
        constexpr int t = only.value;
#pragma unroll 1
        for (int st = s0 + wk; st < s1; st += WK) {
          const bool fresh = st < new_steps;
          const int base = (fresh ? st : st - new_steps) * kStepKeys, end = fresh ? a.nodes : len;
          const int64_t k_step = fresh ? a.kn_node : a.c_slot, v_step = fresh ? a.vn_node : a.c_slot;
          const T* kf = fresh ? static_cast<const T*>(a.k_new) + b * a.kn_row + kvh * a.kn_head : kc;
          const T* vf = fresh ? static_cast<const T*>(a.v_new) + b * a.vn_row + kvh * a.vn_head : vc;
          x[t] = {0.f, 0.f, 0.f, 0.f}, y[t] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            __builtin_amdgcn_sched_barrier(0);
            x[t] = Mma<T>::mma(ld_g16(kf + min(base + step_key(i, 0), end - 1) * k_step + (c * 4 + g) * 8), q[t][c], x[t]);
            y[t] = Mma<T>::mma(ld_g16(kf + min(base + step_key(i, 1), end - 1) * k_step + (c * 4 + g) * 8), q[t][c], y[t]);
          }
          weights(Step{0, base, end, true, fresh, false}, only);
          uint32_t one[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            one[j] = Mma<T>::pack((seen[t] >> (2 * j)) & 1 ? 1.f : 0.f, (seen[t] >> (2 * j + 1)) & 1 ? 1.f : 0.f);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            __builtin_amdgcn_sched_barrier(0);
            const uint16_t* col = reinterpret_cast<const uint16_t*>(vf) + 16 * e + i;
            uint32_t v[4], c[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int key = base + 16 * (w >> 1) + 4 * g + 2 * (w & 1);
              v[w] = (key < end ? ld_g(col + min(key, end - 1) * v_step) : 0u) |
                     (key + 1 < end ? (uint32_t)ld_g(col + min(key + 1, end - 1) * v_step) << 16 : 0u);
              c[w] = F::classes(v[w]), v[w] = F::finite_part(v[w]);
            }
            o[t][e] = Mma<T>::mma(make_uint4(v[0], v[1], v[2], v[3]), ph[t], o[t][e]);
            o[t][e] = Mma<T>::mma(make_uint4(v[0], v[1], v[2], v[3]), pl[t], o[t][e]);
            const f32x4_t sum = Mma<T>::mma(make_uint4(c[0], c[1], c[2], c[3]), make_uint4(one[0], one[1], one[2], one[3]),
                                            f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int r = 0; r < 4; ++r) o[t][e][r] += F::class_value(sum[r]);
          }
        }
      };
      tile(std::integral_constant<int, 0>{});
      if constexpr (NR == 2) tile(std::integral_constant<int, 1>{});
    }
    const int64_t slot = sh.chunk > 0 || a.teams == 0 ? team : (int64_t)b * a.kv_heads + kvh + team;
    // every load into LDS has landed and every stage been read
    __builtin_amdgcn_s_waitcnt(vm_wait_imm(0));
#pragma unroll
    for (int t = 0; t < NR; ++t) l[t] = sum_over_groups(l[t]);
    if constexpr (WK == 1) {
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        const int row = row0 + t * 16 + i;
        if (row >= R) continue;
        const bool there = sees[row / n] != 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float v[4] = {o[t][e][0], o[t][e][1], o[t][e][2], o[t][e][3]};
          emit<T, 4>(a, all, slot, b, kvh, row, 16 * e + 4 * g, v, m[t], l[t], there);
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < NR; ++t)
        if (g == 0) ml[wk][(wr * NR + t) * 16 + i] = make_float2(m[t], l[t]);
      __syncthreads();
      f32x4_t* buf = reinterpret_cast<f32x4_t*>(lds);
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        const int x = (wr * NR + t) * 16 + i;
        float top = ml[0][x].x;
#pragma unroll
        for (int w = 1; w < WK; ++w) top = fmaxf(top, ml[w][x].x);
        const float f = fade(m[t] - top);
#pragma unroll
        for (int e = 0; e < E; ++e) buf[((wid * NR + t) * E + e) * 64 + lane] = o[t][e] * f;
      }
      __syncthreads();
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        const int row = row0 + t * 16 + i, x = (wr * NR + t) * 16 + i;
        if (row >= R) continue;
        float top = ml[0][x].x, sum = 0.f;
#pragma unroll
        for (int w = 1; w < WK; ++w) top = fmaxf(top, ml[w][x].x);
#pragma unroll
        for (int w = 0; w < WK; ++w) sum = fmaf(ml[w][x].y, __builtin_amdgcn_exp2f(ml[w][x].x - top), sum);
        const bool there = sees[row / n] != 0;
        for (int e = wk; e < E; e += WK) {
          f32x4_t u = buf[((wr * NR + t) * E + e) * 64 + lane];
#pragma unroll
          for (int w = 1; w < WK; ++w) u += buf[(((w * WR + wr) * NR + t) * E + e) * 64 + lane];
          const float v[4] = {u[0], u[1], u[2], u[3]};
          emit<T, 4>(a, all, slot, b, kvh, row, 16 * e + 4 * g, v, top, sum, there);
        }
      }
    }
    if (!all && s0 == 0 && rb == 0 && wid == 0) {  // the same from every K/V head
      const uint64_t there = __ballot(sees[lane] != 0);
      if (lane == 0) a.present[b] = there;
    }
    at = unit_at + s1;
    if (s1 == steps) {
      unit_at += steps + kUnitCost;
      if (++kvh == a.kv_heads) kvh = 0, ++b;
    }
    __syncthreads();  // LDS may be written again
  }
}

// Sums the parts of the rows of units that were cut, kJoinRows rows a wave (one where
// there are few: then the latency of a row counts): `cols` lanes
// share the dimensions, the others further parts.
template <typename T, int kJoinRows>
__global__ __launch_bounds__(256) void k_tree_join(const TreeArgs a, bool many, int cols) {
  const int lane = threadIdx.x & 63, n = a.heads / a.kv_heads, R = a.nodes * n;
  const int blocks = (R + 4 * kJoinRows - 1) / (4 * kJoinRows), unit = blockIdx.x / blocks;
  const int r0 = ((blockIdx.x - unit * blocks) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kJoinRows;
  if (r0 >= R) return;
  const int b = unit / a.kv_heads, kvh = unit - b * a.kv_heads;
  int64_t first = 0;
  int parts = 0;
  const int steps = steps_of(a, b);
  if (a.teams == 0) {
    const int chunk = own_chunk(a, steps);
    parts = (steps + chunk - 1) / chunk;
    first = (int64_t)unit * a.splits;
  } else {
    const Share sh = share_of(a, lane);
    const int chunk = sh.chunk > 0 ? sh.chunk : many ? 0 : (int)((sh.total + a.teams - 1) / a.teams);
    int64_t before = 0;  // parts, or steps, of the sequences before
    for (int x = lane; x < b; x += 64) before += chunk > 0 ? (steps_of(a, x) + chunk - 1) / chunk : kUnitCost + steps_of(a, x);
    before = wave_sum64(before) * a.kv_heads;
    if (chunk > 0) {
      parts = (steps + chunk - 1) / chunk;
      first = before + (int64_t)kvh * parts;
    } else {
      const int64_t at = before + (int64_t)kvh * (kUnitCost + steps) + kUnitCost, t0 = team_of(sh, a.teams, at);
      parts = (int)(team_of(sh, a.teams, at + steps - 1) - t0) + 1;
      first = unit + t0;
    }
  }
  if (parts == 1) return;  // written by its block
  const uint64_t present = a.present[b];
  const int d = lane % cols * 4, from = lane / cols, every = 64 / cols;
#pragma unroll
  for (int x = 0; x < kJoinRows; ++x) {
    const int r = r0 + x;
    if (r >= R) break;
    const float2* ml = a.part_ml + first * R + r;
    const float* part = a.part + (first * R + r) * a.D;
    float top = kNone, sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < parts; s0 += 64) {
      const float2 y = s0 + lane < parts ? ml[(size_t)(s0 + lane) * R] : make_float2(kNone, 0.f);
      const float to = fmaxf(top, wave_max(y.x)), f = fade(top - to);
      top = to;
      const float w = s0 + lane < parts ? fade(y.x - top) : 0.f;
      sum = fmaf(sum, f, wave_sum(y.y * w));
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= f;
      const int end = min(64, parts - s0);
      for (int s = from; s < ((end + every - 1) / every) * every; s += every) {
        const float ws = __shfl(w, s, 64);
        if (s < end && d < a.D) {
          const float4 z = *reinterpret_cast<const float4*>(part + (size_t)(s0 + s) * R * a.D + d);
          v[0] = fmaf(z.x, ws, v[0]), v[1] = fmaf(z.y, ws, v[1]), v[2] = fmaf(z.z, ws, v[2]), v[3] = fmaf(z.w, ws, v[3]);
        }
      }
    }
    for (int o = cols; o < 64; o <<= 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += __shfl_xor(v[e], o, 64);
    }
    const int node = r / n, h = kvh * n + r - node * n;
    const bool there = ((present >> node) & 1) && sum != 0.f;
    const float inv = 1.f / sum;
    if (d < a.D && from == 0) {
      T* dst = static_cast<T*>(a.out) + b * a.o_row + node * a.o_node + h * a.o_head + d;
      union {
        T x[4];
        uint4 w4;
        uint2 w2;
      } u;
#pragma unroll
      for (int e = 0; e < 4; ++e) u.x[e] = St<T>::st(there ? v[e] * inv : 0.f);
      if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst) = u.w4;
      else *reinterpret_cast<uint2*>(dst) = u.w2;
    }
    if (a.lse != nullptr && lane == 0)
      a.lse[((size_t)b * a.nodes + node) * a.heads + h] = there ? fmaf(top, kLn2, logf(sum)) : -INFINITY;
  }
}

// Row tiles that a wave of k_tree_few holds: the output takes dp / 4 registers a tile,
// queries as much again in 16-bit types (twice that in fp32), a step's keys and values dp / 2.
constexpr int row_tiles(size_t elt, int dp) {
  return dp == 256 ? 1 : elt == 4 || dp == 128 ? 2 : 4;
}

struct Plan {
  bool many;
  int tiles;  // row tiles of a block
  int row_blocks, teams, splits, least;
};

Plan plan(const KvCache& c, int heads, int nodes) {
  const int R = nodes * (heads / c.kv_heads), dp = c.d <= 32 ? 32 : c.d <= 64 ? 64 : c.d <= 128 ? 128 : 256;
  Plan p;
  // Times in us, bf16, 4 sequences, 8 K/V heads, d 128 unless said otherwise.
  // 24 rows, 16384 entries: 61 by k_tree_many, 103 by k_tree_few; 16 rows 61 and 58.
  // Row tiles 2 / 4 / 8 / 16 over 8192 entries: 64 rows 47 / 41 / 49 / 69, 256 rows
  // 111 / 85 / 84 / 79.
  p.many = R > 16 && c.dt != DType::F32 && (c.d == 64 || c.d == 128);
  p.tiles = p.many ? (R <= 32 ? 2 : R <= 64 ? 4 : R <= 128 ? 8 : 16)
                   : std::min(row_tiles(dtype_size(c.dt), dp), R <= 16 ? 1 : R <= 32 ? 2 : 4);
  p.row_blocks = (R + 16 * p.tiles - 1) / (16 * p.tiles);
  const int64_t steps = (c.capacity + kStepKeys - 1) / kStepKeys + (nodes + kStepKeys - 1) / kStepKeys;
  const int64_t units = std::max<int64_t>(1, (int64_t)c.rows * c.kv_heads);
  // k_tree_many fills a CU with a block (128 / 256 / 512 teams for 64 rows, 16384 entries:
  // 76 / 64 / 76), of k_tree_few a CU holds two (256 / 512 / 1024 parts for one node: 60 / 58 /
  // 62).  Parts of 8 steps at least: one node over 1000 entries, d 64, with 4 / 8 / 16 / 32
  // steps 11.5 / 11.6 / 13.3 / 19.1.
  // Up to 32768 steps the units are cut by themselves: 300 sequences of 2048, one K/V head,
  // 76 against 95 shared out by all lengths (k_tree_few), 51 against 58 (k_tree_many, d 64).
  // Beyond, unequal lengths would cost more than that: 32 sequences of 100 and one of 8192,
  // one node, 25 shared out and 71 by themselves (32 of 8192: 191 and 186).
  p.least = 8;
  p.splits = 1;
  p.teams = std::max(8, (p.many ? 256 : 512) / p.row_blocks / 8 * 8);
  if (steps * units * p.row_blocks <= 32768) {
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>((steps + p.least - 1) / p.least, p.teams / units));
    p.teams = 0;
  }
  return p;
}

bool cuts(const Plan& p) { return p.teams > 0 || p.splits > 1; }
size_t blocks_of(const KvCache& c, const Plan& p) {  // and slots, where units are cut
  const size_t units = (size_t)c.rows * c.kv_heads;
  return p.teams > 0 ? p.teams + units : units * p.splits;
}

// Rows that a wave of k_tree_join takes: 1056 rows 16.1 us by ones and 21.2 by fours, with the
// attention, 32768 rows 232 and 228.
int join_rows(int64_t units, int R) { return units * R < 16384 ? 1 : 4; }

template <typename T, int DP, int NR>
void launch_few(const TreeArgs& a, int blocks, hipStream_t s) {
  const size_t join = (size_t)kWaves * NR * AttnFrag<T, DP>::E * 64 * 16;
  const size_t lds = std::max(join, a.bias != nullptr ? (size_t)kBiasLds * 4 : size_t{0});
  allow_dynamic_lds(reinterpret_cast<const void*>(&k_tree_few<T, DP, NR>), std::max(join, (size_t)kBiasLds * 4));
  hipLaunchKernelGGL((k_tree_few<T, DP, NR>), dim3(blocks * a.row_blocks), dim3(64 * kWaves), lds, s, a);
}

template <typename T, int DP>
void launch_few(const TreeArgs& a, int blocks, int nr, hipStream_t s) {
  constexpr int most = row_tiles(sizeof(T), DP);
  if (nr == 1) return launch_few<T, DP, 1>(a, blocks, s);
  if constexpr (most >= 2)
    if (nr == 2) return launch_few<T, DP, 2>(a, blocks, s);
  if constexpr (most >= 4) launch_few<T, DP, 4>(a, blocks, s);
}

template <typename T, int DP, int WR, int NR>
void launch_many(const TreeArgs& a, int blocks, hipStream_t s) {
  using M = Many<DP, WR, NR>;
  const dim3 grid((blocks + 7) / 8 * 8 * a.row_blocks);
  if (a.bias != nullptr) {
    const size_t lds = M::kLds + (size_t)kBiasLds * 4;
    allow_dynamic_lds(reinterpret_cast<const void*>(&k_tree_many<T, DP, WR, NR, true>), lds);
    hipLaunchKernelGGL((k_tree_many<T, DP, WR, NR, true>), grid, dim3(512), lds, s, a);
  } else {
    allow_dynamic_lds(reinterpret_cast<const void*>(&k_tree_many<T, DP, WR, NR, false>), M::kLds);
    hipLaunchKernelGGL((k_tree_many<T, DP, WR, NR, false>), grid, dim3(512), M::kLds, s, a);
  }
}

template <typename T, int DP>
void launch_many(const TreeArgs& a, int blocks, int tiles, hipStream_t s) {
  if (tiles == 2) launch_many<T, DP, 2, 1>(a, blocks, s);
  else if (tiles == 4) launch_many<T, DP, 4, 1>(a, blocks, s);
  else if (tiles == 8) launch_many<T, DP, 8, 1>(a, blocks, s);
  else launch_many<T, DP, 8, 2>(a, blocks, s);
}

}  // namespace

bool tree_attention_fits(const KvCache& c, int heads, int nodes) {
  const Plan p = plan(c, heads, nodes);
  const int64_t units = (int64_t)c.rows * c.kv_heads, most = (1ll << 32) - 1;  // threads of a launch
  const int R = nodes * (heads / c.kv_heads), per = 4 * join_rows(units, R);
  const int64_t blocks = ((int64_t)blocks_of(c, p) + 7) / 8 * 8 * p.row_blocks;
  return blocks * (p.many ? 512 : 64 * kWaves) <= most && units * ((R + per - 1) / per) * 256 <= most;
}

size_t tree_attention_workspace(const KvCache& c, int heads, int nodes) {
  const Plan p = plan(c, heads, nodes);
  if (!cuts(p)) return 0;
  return blocks_of(c, p) * (size_t)(heads / c.kv_heads * nodes) * (c.d + 2) * 4 + (size_t)c.rows * 8;
}

void tree_attention(const KvCache& c, const TreeAttnArgs& t, void* ws, hipStream_t s) {
  const Plan p = plan(c, t.heads, t.nodes);
  TreeArgs a{};
  a.q = t.q.p, a.k_new = t.k_new.p, a.v_new = t.v_new.p, a.k = c.k, a.v = c.v, a.out = t.out.p;
  a.parents = t.parents, a.length = c.length, a.pos = c.pos, a.next_pos = c.pos != nullptr ? c.next_pos : nullptr;
  a.bias = t.bias, a.lse = t.lse;
  a.q_row = t.q.row_stride, a.q_node = t.q.node_stride, a.q_head = t.q.head_stride;
  a.kn_row = t.k_new.row_stride, a.kn_node = t.k_new.node_stride, a.kn_head = t.k_new.head_stride;
  a.vn_row = t.v_new.row_stride, a.vn_node = t.v_new.node_stride, a.vn_head = t.v_new.head_stride;
  a.o_row = t.out.row_stride, a.o_node = t.out.node_stride, a.o_head = t.out.head_stride;
  a.c_row = c.row_stride, a.c_head = c.head_stride, a.c_slot = c.slot_stride, a.parents_stride = t.parents_stride;
  a.rows = c.rows, a.capacity = c.capacity, a.kv_heads = c.kv_heads, a.heads = t.heads, a.nodes = t.nodes, a.D = c.d;
  a.buckets = t.buckets, a.teams = p.teams, a.splits = p.splits, a.least = p.least, a.row_blocks = p.row_blocks;
  a.scale = t.scale;
  const int R = t.nodes * (t.heads / c.kv_heads);
  if (cuts(p)) {
    const size_t rows = blocks_of(c, p) * R;
    a.part = static_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(a.part + rows * c.d);
    a.present = reinterpret_cast<uint64_t*>(a.part_ml + rows);
  }
  const int blocks = (int)blocks_of(c, p);
  if (p.many) {
    auto go = [&](auto x) {
      using T = decltype(x);
      if (c.d == 64) launch_many<T, 64>(a, blocks, p.tiles, s);
      else launch_many<T, 128>(a, blocks, p.tiles, s);
    };
    if (c.dt == DType::BF16) go(bf16{});
    else go(f16{});
  } else {
    MRT_DTYPE_DISPATCH(c.dt, {
      if (c.d <= 32) launch_few<T, 32>(a, blocks, p.tiles, s);
      else if (c.d <= 64) launch_few<T, 64>(a, blocks, p.tiles, s);
      else if (c.d <= 128) launch_few<T, 128>(a, blocks, p.tiles, s);
      else launch_few<T, 256>(a, blocks, p.tiles, s);
    });
  }
  MRT_HIP_CHECK(hipGetLastError());
  if (cuts(p)) {
    const int cols = c.d <= 32 ? 8 : c.d <= 64 ? 16 : c.d <= 128 ? 32 : 64, units = c.rows * c.kv_heads;
    MRT_DTYPE_DISPATCH(c.dt, {
      if (join_rows(units, R) == 1)
        hipLaunchKernelGGL((k_tree_join<T, 1>), dim3(units * ((R + 3) / 4)), dim3(256), 0, s, a, p.many, cols);
      else
        hipLaunchKernelGGL((k_tree_join<T, 4>), dim3(units * ((R + 15) / 16)), dim3(256), 0, s, a, p.many, cols);
    });
    MRT_HIP_CHECK(hipGetLastError());
  }
}

}  // namespace mrt
