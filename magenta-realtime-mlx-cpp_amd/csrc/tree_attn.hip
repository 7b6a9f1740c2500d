// Attention of a tree of drafted tokens over a cache.
//
// Node t of a sequence (parent -1: follows the cache; else an earlier node) attends
// every cache entry, its ancestors and itself:
//   s_tj = scale q_t . k_j + bias[h, min(distance, M - 1)],  out_t = softmax(s_t) V.
// One pass over the keys with the running maximum and sum of the softmax.
//
// Work split: the n = heads / kv_heads query heads of a KV head share its keys, so a
// KV head's rows are r = t n + hq, R = nodes n of them, 16 NR to a block; the keys are
// cut into splits, a block each, whose four waves take steps of 32 keys in turn, each
// with its own maximum, sum and output in registers (attn_frag.hpp).  The drafted
// nodes are the last steps of a sequence.  Blocks of one split write the output; with
// more, each leaves (maximum, sum, output) in fp32 and k_tree_join sums them in order,
// so a result does not depend on timing.
#include <algorithm>
#include <type_traits>

#include "attn_frag.hpp"
#include "kv_cache.hpp"
#include "mfma_ring.hpp"

namespace mrt {
namespace {

constexpr int kWaves = 4;
constexpr float kNone = -1e30f;  // running maximum before any key: finite, so exp2(-inf - kNone) is 0
constexpr int kBiasLds = 8192;   // floats of the bias by distance kept in LDS

struct TreeArgs {
  const void *q, *k_new, *v_new, *k, *v;
  void* out;
  const int *parents, *length, *pos, *next_pos;
  const float* bias;
  float* lse;
  float* part;        // (rows * kv_heads, splits, R, D) outputs of the splits
  float2* part_ml;    // (rows * kv_heads, splits, R) maximum (in log2 units) and sum
  uint64_t* present;  // (rows) mask of the nodes that are there
  int64_t q_row, q_node, q_head, kn_row, kn_node, kn_head, vn_row, vn_node, vn_head, o_row, o_node, o_head;
  int64_t c_row, c_head, c_slot, parents_stride;
  int capacity, kv_heads, heads, nodes, D, buckets, splits, split_steps, row_blocks, units;
  float scale;
};

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

template <typename T, int DP, int NR>
__global__ __launch_bounds__(64 * kWaves, 1) void k_tree(const TreeArgs a) {
  using F = AttnFrag<T, DP>;
  constexpr int E = F::E, VW = F::VW, KC = F::KC;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4, D = a.D;
  // Row blocks of the same keys follow each other on one XCD, whose L2 they share.
  const int id = blockIdx.x >> 3, unit = (id / a.row_blocks) * 8 + (blockIdx.x & 7);
  if (unit >= a.units) return;
  const int row0 = (id % a.row_blocks) * (16 * NR);
  const int bg = unit / a.splits, split = unit - bg * a.splits;
  const int b = bg / a.kv_heads, kvh = bg - b * a.kv_heads, n = a.heads / a.kv_heads, R = a.nodes * n;
  const int len = min(max(a.length[b], 0), a.capacity);
  const int old_steps = (len + kStepKeys - 1) / kStepKeys;
  const int steps = old_steps + (a.nodes + kStepKeys - 1) / kStepKeys;
  const int s0 = split * a.split_steps, s1 = min(steps, s0 + a.split_steps);
  if (s0 >= steps) return;

  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ uint64_t sees[kMaxNodes];
  __shared__ float2 ml[kWaves][16 * NR];
  float* btab = reinterpret_cast<float*>(lds);  // the bias of this KV head's heads, until the waves join
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
  __syncthreads();

  const T* kc = static_cast<const T*>(a.k) + b * a.c_row + kvh * a.c_head;
  const T* vc = static_cast<const T*>(a.v) + b * a.c_row + kvh * a.c_head;
  const int* pos = a.pos == nullptr ? nullptr : a.pos + (size_t)bg * a.capacity;
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
#pragma unroll
  for (int t = 0; t < NR; ++t) {
    m[t] = kNone, l[t] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[t][e] = {0.f, 0.f, 0.f, 0.f};
  }
  const float scale2 = a.scale * kLog2e;
  // m is the maximum less kShift: fp16 weights reach up to 2^15, so that those far
  // below the maximum keep their bits.
  constexpr float kShift = std::is_same_v<T, f16> ? 15.f : 0.f;

  for (int st = s0 + wid; st < s1; st += kWaves) {
    const bool fresh = st >= old_steps;  // drafted nodes
    const int base = (fresh ? st - old_steps : st) * kStepKeys, end = fresh ? a.nodes : len;
    const T* kb = fresh ? static_cast<const T*>(a.k_new) + b * a.kn_row + kvh * a.kn_head : kc;
    const T* vb = fresh ? static_cast<const T*>(a.v_new) + b * a.vn_row + kvh * a.vn_head : vc;
    const int64_t kstep = fresh ? a.kn_node : a.c_slot, vstep = fresh ? a.vn_node : a.c_slot;
    const bool whole = base + kStepKeys <= end;
    uint4 kf[2][KC];
    uint32_t vf[8][VW];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      F::load_row(kb + (int64_t)min(base + step_key(i, h), end - 1) * kstep, g, D, kf[h]);
#pragma unroll
    for (int j = 0; j < 8; ++j) F::load_v(vb + (int64_t)min(base + 8 * g + j, end - 1) * vstep, i, D, vf[j]);
    if (!whole) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int w = 0; w < VW; ++w) vf[j][w] = base + 8 * g + j < end ? vf[j][w] : 0u;
    }
    float p[NR][8];
    int kpos[8];
    if (a.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = min(base + 8 * g + j, end - 1);
        kpos[j] = fresh ? __popcll(sees[key]) - 1 : pos != nullptr ? pos[key] : key;
      }
    }
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      const f32x4_t x = F::scores(kf[0], q[t]), y = F::scores(kf[1], q[t]);
      float s[8] = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      if (a.bias != nullptr) {
        const int at = fresh ? __popcll(sees[min(row0 + t * 16 + i, R - 1) / n]) - 1 : qpos[t];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          s[j] = fmaf(s[j], scale2, brow[t][min(max(at - kpos[j], 0), a.buckets - 1)] * kLog2e);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] *= scale2;
      }
      if (fresh) {
        const uint64_t see = sees[min(row0 + t * 16 + i, R - 1) / n] >> base;
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = (see >> (8 * g + j)) & 1 ? s[j] : -INFINITY;
      } else if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = base + 8 * g + j < end ? s[j] : -INFINITY;
      }
      float top = s[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) top = fmaxf(top, s[j]);
      top = max_over_groups(top) - kShift;
      if (__any(top > m[t])) {
        const float mn = fmaxf(m[t], top), f = __builtin_amdgcn_exp2f(m[t] - mn);
        m[t] = mn;
        l[t] *= f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[t][e] *= f;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[t][j] = __builtin_amdgcn_exp2f(s[j] - m[t]);
        l[t] += p[t][j];
      }
    }
    if (!fresh) {
      F::template add_pv<NR>(vf, p, o);
    } else {
      // A node's infinities and NaN belong to those who see it: 0 * inf is NaN in a
      // matrix product, so they are left out of it and added by class.
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
      if (__any(diff != 0)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int key = base + 8 * g + j;
          F::load_v(vb + (int64_t)min(key, end - 1) * vstep, i, D, vf[j]);
#pragma unroll
          for (int w = 0; w < VW; ++w) vf[j][w] = key < end ? F::classes(vf[j][w]) : 0u;
        }
#pragma unroll
        for (int t = 0; t < NR; ++t) {
          const uint64_t see = sees[min(row0 + t * 16 + i, R - 1) / n] >> base;
          float one[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) one[j] = (see >> (8 * g + j)) & 1 ? 1.f : 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const f32x4_t c = F::count(vf, one, e);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[t][e][r] += F::class_value(c[r]);
          }
        }
      }
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
    const float f = __builtin_amdgcn_exp2f(m[t] - top);
#pragma unroll
    for (int e = 0; e < E; ++e) buf[((wid * NR + t) * E + e) * 64 + lane] = o[t][e] * f;
  }
  __syncthreads();
  // Thread (lane, r = wid): dimensions (4 g + r) E .. + E - 1 of row i of each tile.
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
    const int node = r / n, h = kvh * n + r - node * n;
    if (a.splits == 1) {
      const bool there = sees[node] != 0;
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
          if (d + w * (int)(16 / sizeof(T)) < D) reinterpret_cast<uint4*>(dst)[w] = u.w4[w];
      } else if (d < D) {
        if constexpr (E * sizeof(T) == 8) *reinterpret_cast<uint2*>(dst) = u.w2;
        else *reinterpret_cast<uint32_t*>(dst) = u.w1;
      }
      if (a.lse != nullptr && d == 0)
        a.lse[((size_t)b * a.nodes + node) * a.heads + h] = there ? fmaf(top, kLn2, logf(sum)) : -INFINITY;
    } else {
      const size_t at = ((size_t)bg * a.splits + split) * R + r;
      float* dst = a.part + at * D + d;
#pragma unroll
      for (int e = 0; e < E; e += 2)
        if (d + e < D) *reinterpret_cast<float2*>(dst + e) = make_float2(v[e], v[e + 1]);
      if (d == 0) a.part_ml[at] = make_float2(top, sum);
    }
  }
  if (a.splits > 1 && s1 > old_steps && kvh == 0 && row0 == 0 && wid == 0) {
    const uint64_t there = __ballot(sees[lane] != 0);
    if (lane == 0) a.present[b] = there;
  }
}

// Sums the splits of one row: a wave a row, each lane some of its dimensions.
template <typename T>
__global__ __launch_bounds__(256) void k_tree_join(const TreeArgs a) {
  const int lane = threadIdx.x & 63, n = a.heads / a.kv_heads, R = a.nodes * n;
  const int blocks = (R + 3) / 4, bg = blockIdx.x / blocks;
  const int r = (blockIdx.x - bg * blocks) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (r >= R) return;
  const int b = bg / a.kv_heads, kvh = bg - b * a.kv_heads, node = r / n, h = kvh * n + r - node * n;
  const int len = min(max(a.length[b], 0), a.capacity);
  const int steps = (len + kStepKeys - 1) / kStepKeys + (a.nodes + kStepKeys - 1) / kStepKeys;
  const int splits = (steps + a.split_steps - 1) / a.split_steps;
  const float2* ml = a.part_ml + (size_t)bg * a.splits * R + r;
  float top = kNone;
  for (int s = lane; s < splits; s += 64) top = fmaxf(top, ml[(size_t)s * R].x);
  top = wave_max(top);
  const float* part = a.part + ((size_t)bg * a.splits * R + r) * a.D;
  float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
  const int d = lane * 4;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float2 x = ml[(size_t)s * R];
    const float f = __builtin_amdgcn_exp2f(x.x - top);
    sum = fmaf(x.y, f, sum);
    if (d < a.D) {
      const float4 y = *reinterpret_cast<const float4*>(part + (size_t)s * R * a.D + d);
      v[0] = fmaf(y.x, f, v[0]), v[1] = fmaf(y.y, f, v[1]), v[2] = fmaf(y.z, f, v[2]), v[3] = fmaf(y.w, f, v[3]);
    }
  }
  const bool there = (a.present[b] >> node) & 1;
  const float inv = 1.f / sum;
  if (d < a.D) {
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

// Row tiles that a wave's registers hold: the output takes dp / 4 a tile, queries as
// much again in 16-bit types (twice that in fp32), a step's keys and values dp / 2.
constexpr int row_tiles(size_t elt, int dp) {
  return dp == 256 ? 1 : elt == 4 || dp == 128 ? 2 : 4;
}

struct Plan {
  int nr, splits, split_steps, row_blocks;
};

Plan plan(const KvCache& c, int heads, int nodes) {
  const int R = nodes * (heads / c.kv_heads), dp = c.d <= 32 ? 32 : c.d <= 64 ? 64 : c.d <= 128 ? 128 : 256;
  const int most = row_tiles(dtype_size(c.dt), dp);
  Plan p;
  p.nr = std::min(most, R <= 16 ? 1 : R <= 32 ? 2 : 4);
  p.row_blocks = (R + 16 * p.nr - 1) / (16 * p.nr);
  const int steps = (c.capacity + kStepKeys - 1) / kStepKeys + (nodes + kStepKeys - 1) / kStepKeys;
  const int units = std::max(1, c.rows * c.kv_heads * p.row_blocks);
  const int want = std::max(1, 1024 / units);
  p.split_steps = std::max(2 * kWaves, (steps + want - 1) / want);
  p.splits = (steps + p.split_steps - 1) / p.split_steps;
  if (p.splits == 1) p.split_steps = steps;
  return p;
}

template <typename T, int DP, int NR>
void launch(const TreeArgs& a, hipStream_t s) {
  const size_t join = (size_t)kWaves * NR * AttnFrag<T, DP>::E * 64 * 16;
  const size_t lds = std::max(join, a.bias != nullptr ? (size_t)kBiasLds * 4 : size_t{0});
  allow_dynamic_lds(reinterpret_cast<const void*>(&k_tree<T, DP, NR>), std::max(join, (size_t)kBiasLds * 4));
  const int grid = (a.units + 7) / 8 * 8 * a.row_blocks;
  hipLaunchKernelGGL((k_tree<T, DP, NR>), dim3(grid), dim3(64 * kWaves), lds, s, a);
}

template <typename T, int DP>
void launch_nr(const TreeArgs& a, int nr, hipStream_t s) {
  constexpr int most = row_tiles(sizeof(T), DP);
  if (nr == 1) return launch<T, DP, 1>(a, s);
  if constexpr (most >= 2)
    if (nr == 2) return launch<T, DP, 2>(a, s);
  if constexpr (most >= 4) launch<T, DP, 4>(a, s);
}

}  // namespace

size_t tree_attention_workspace(const KvCache& c, int heads, int nodes) {
  const Plan p = plan(c, heads, nodes);
  if (p.splits == 1) return 0;
  const size_t rows = (size_t)c.rows * heads * nodes * p.splits;
  return rows * (c.d + 2) * 4 + (size_t)c.rows * 8;
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
  a.capacity = c.capacity, a.kv_heads = c.kv_heads, a.heads = t.heads, a.nodes = t.nodes, a.D = c.d;
  a.buckets = t.buckets, a.splits = p.splits, a.split_steps = p.split_steps, a.row_blocks = p.row_blocks;
  a.units = c.rows * c.kv_heads * p.splits;
  a.scale = t.scale;
  if (p.splits > 1) {
    const size_t rows = (size_t)c.rows * t.heads * t.nodes * p.splits;
    a.part = static_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(a.part + rows * c.d);
    a.present = reinterpret_cast<uint64_t*>(a.part_ml + rows);
  }
  MRT_DTYPE_DISPATCH(c.dt, {
    if (c.d <= 32) launch_nr<T, 32>(a, p.nr, s);
    else if (c.d <= 64) launch_nr<T, 64>(a, p.nr, s);
    else if (c.d <= 128) launch_nr<T, 128>(a, p.nr, s);
    else launch_nr<T, 256>(a, p.nr, s);
  });
  MRT_HIP_CHECK(hipGetLastError());
  if (p.splits > 1) {
    const int R = t.nodes * (t.heads / c.kv_heads);
    const dim3 grid(c.rows * c.kv_heads * ((R + 3) / 4));
    MRT_DTYPE_DISPATCH(c.dt, hipLaunchKernelGGL(k_tree_join<T>, grid, dim3(256), 0, s, a));
    MRT_HIP_CHECK(hipGetLastError());
  }
}

}  // namespace mrt
