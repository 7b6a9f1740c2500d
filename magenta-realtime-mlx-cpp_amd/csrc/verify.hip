// Verification of a tree of drafted tokens: which path of it the target's probabilities
// accept, by given random numbers, and the token that follows.
//
// At a slot with target p and draft q, its children in order (r_0 = p, Z_0 = 1):
//   child j with token x is accepted if u_j Z q(x) < r(x), else r <- max(r - Z q, 0), Z <- sum r,
// and if none is, the token is drawn from r: the first whose sum of r up to it exceeds
// u sum r.  Where children were drawn from q one by one, the tokens have the target's own
// distribution.  Without q (drafts that were not drawn): u_j Z < r(x), else r(x) <- 0, Z <- Z - r(x).
//
// All of it in 64 bits: a drawn token is a comparison of sums over the vocabulary, and with sums
// in 32 bits it would depend on their order.
//
// A block a sequence.  Each node's own p(x) and q(x) are gathered at once, so tests need no
// memory; a rejection costs one pass over the slot's rows, in which wave w sums segments w,
// w + 16, ..; the drawn token's segment is the only one looked at again.
#include <algorithm>

#include "device_utils.hpp"
#include "verify.hpp"

namespace mrt {
namespace {

constexpr int kWaves = 16;
constexpr int kSegments = 256;

// What is not a positive finite number counts as 0.
__device__ __forceinline__ float counted(float p) { return p > 0.f && p < INFINITY ? p : 0.f; }

// VEC consecutive probabilities; 0 past the end.
template <typename T, int VEC>
__device__ __forceinline__ uint4 load_raw(const T* row, int at, int V, bool wide) {
  if (wide && at + VEC <= V) return ld_g16(row + at);
  union {
    T x[VEC];
    uint4 w;
  } u;
#pragma unroll
  for (int e = 0; e < VEC; ++e) u.x[e] = at + e < V ? ld_g(row + at + e) : T(0);
  return u.w;
}
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const uint4& w, float (&x)[VEC]) {
  union {
    uint4 w;
    T x[VEC];
  } u;
  u.w = w;
#pragma unroll
  for (int e = 0; e < VEC; ++e) x[e] = counted(St<T>::ld(u.x[e]));
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

struct Rejections {
  double z[kMaxNodes + 1];  // Z before each rejection
  int token[kMaxNodes];     // the rejected tokens
};

// r of element `at` after n rejections.
template <bool DRAFT>
__device__ __forceinline__ double rest(double p, double q, int at, const Rejections& j, int n) {
  for (int k = 0; k < n; ++k) {
    if constexpr (DRAFT) p = fmax(p - j.z[k] * q, 0.0);
    else p = at == j.token[k] ? 0.0 : p;
  }
  return p;
}

template <typename T, bool DRAFT>
__global__ __launch_bounds__(64 * kWaves) void k_verify(const VerifyArgs a, bool wide) {
  constexpr int VEC = 16 / sizeof(T), CHUNK = 64 * VEC;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int N = a.nodes, V = a.vocab;
  __shared__ double own_p[kMaxNodes], own_q[kMaxNodes], own_u[kMaxNodes + 1];
  __shared__ int parent[kMaxNodes], token[kMaxNodes], path[kMaxNodes];
  __shared__ Rejections rej;
  __shared__ double seg[kSegments];
  __shared__ double total;
  const T* target = static_cast<const T*>(a.target) + b * a.t_row;
  const T* draft = static_cast<const T*>(a.draft) + b * a.d_row;
  if (tid < N) {
    const int up = a.parents != nullptr ? a.parents[b * a.parents_stride + tid] : tid - 1;
    const int x = a.tokens[(int64_t)b * N + tid];
    const bool there = up >= -1 && up < tid, known = x >= 0 && x < V;
    parent[tid] = there ? up : -2;
    token[tid] = known ? x : -1;
    own_p[tid] = there && known ? (double)counted(St<T>::ld(target[(up + 1) * a.t_slot + x])) : 0.0;
    own_q[tid] = DRAFT && there && known ? (double)counted(St<T>::ld(draft[(up + 1) * a.d_slot + x])) : 1.0;
  }
  if (tid <= N) own_u[tid] = a.uniforms[(int64_t)b * (N + 1) + tid];
  __syncthreads();

  const int chunks = (V + CHUNK - 1) / CHUNK, per = (chunks + kSegments - 1) / kSegments;
  const int segments = (chunks + per - 1) / per;
  // The sums of r after n rejections at slot s: of each segment, running, and of all.
  auto pass = [&](int s, int n) {
    const T* p = target + s * a.t_slot;
    const T* q = draft + s * a.d_slot;
    const bool both = DRAFT && n > 0;
    for (int x = wid; x < segments; x += kWaves) {
      double sum = 0.0;
      const int end = min((x + 1) * per, chunks);
      for (int c = x * per; c < end; ++c) {
        const int at = c * CHUNK + lane * VEC;
        float pv[VEC], qv[VEC];
        unpack<T, VEC>(load_raw<T, VEC>(p, at, V, wide), pv);
        if (both) unpack<T, VEC>(load_raw<T, VEC>(q, at, V, wide), qv);
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum += rest<DRAFT>((double)pv[e], both ? (double)qv[e] : 0.0, at + e, rej, n);
      }
      sum = wave_sum(sum);
      if (lane == 0) seg[x] = sum;
    }
    __syncthreads();
    if (wid == 0) {  // running sums, four segments a lane
      double v[4], run = 0.0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        run += lane * 4 + k < segments ? seg[lane * 4 + k] : 0.0;
        v[k] = run;
      }
      double incl = run;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double y = __shfl_up(incl, o, 64);
        if (lane >= o) incl += y;
      }
      double before = __shfl_up(incl, 1, 64);
      if (lane == 0) before = 0.0;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (lane * 4 + k < segments) seg[lane * 4 + k] = before + v[k];
      if (lane == 63) total = incl;
    }
    __syncthreads();
  };

  // The path, the same in every thread.
  int here = 0, n = 0, count = 0;  // slot, rejections there, accepted nodes
  bool summed = false;             // the last pass was of this slot and n
  double z = 1.0;
  for (int t = 0; t < N; ++t) {
    if (parent[t] + 1 != here) continue;
    const int x = token[t];
    if (x < 0) continue;  // not a token: nothing was drawn
    if (DRAFT && n > 0 && !summed) {
      pass(here, n);
      summed = true;
      z = total;
    }
    const double r = rest<DRAFT>(own_p[t], own_q[t], x, rej, n);
    if (own_u[t] * z * own_q[t] < r) {
      if (tid == 0) path[count] = t;
      ++count;
      here = t + 1, n = 0, z = 1.0, summed = false;
    } else {
      __syncthreads();  // everyone has read what is there
      if (tid == 0) rej.z[n] = z, rej.token[n] = x;
      __syncthreads();
      if (!DRAFT) z -= r;
      ++n;
      summed = false;
    }
  }
  if (!summed) pass(here, n);
  if (!(total > 0.0) && n > 0) {  // nothing left: the target itself
    __syncthreads();
    n = 0;
    pass(here, 0);
  }
  if (tid < N) a.accepted[(int64_t)b * N + tid] = tid < count ? path[tid] : -1;
  if (tid == 0) a.count[b] = count;
  if (wid != 0) return;

  // The first segment that exceeds the threshold, then its first chunk, lane, token.
  const double sum = total, want = fmax(own_u[N] * sum, 0.0);
  int found = -1;
  for (int s0 = 0; s0 < segments && found < 0; s0 += 64) {
    const uint64_t past = __ballot(s0 + lane < segments && seg[s0 + lane] > want);
    if (past != 0) found = s0 + __ffsll((unsigned long long)past) - 1;
  }
  int drawn = -1, latest = -1;  // latest: the last token with a positive r seen
  const T* p = target + here * a.t_slot;
  const T* q = draft + here * a.d_slot;
  const bool both = DRAFT && n > 0;
  // Without one (a random number of 1): the last token with any weight, over all segments.
  int c = found < 0 ? 0 : found * per;
  const int end = found < 0 ? chunks : min((found + 1) * per, chunks);
  double before = found > 0 ? seg[found - 1] : 0.0;
  for (; c < end && sum > 0.0; ++c) {
    const int at = c * CHUNK + lane * VEC;
    float pv[VEC], qv[VEC];
    unpack<T, VEC>(load_raw<T, VEC>(p, at, V, wide), pv);
    if (both) unpack<T, VEC>(load_raw<T, VEC>(q, at, V, wide), qv);
    double v[VEC], run = 0.0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      v[e] = rest<DRAFT>((double)pv[e], both ? (double)qv[e] : 0.0, at + e, rej, n);
      run += v[e];
    }
    double incl = run;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(incl, o, 64);
      if (lane >= o) incl += y;
    }
    double sofar = __shfl_up(incl, 1, 64);
    if (lane == 0) sofar = 0.0;
    sofar += before;
    int mine = -1, last = -1;  // this lane's first token past the threshold, and last with weight
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sofar += v[e];
      if (v[e] > 0.0) {
        last = at + e;
        if (mine < 0 && sofar > want) mine = at + e;
      }
    }
    const uint64_t any = __ballot(last >= 0), past = __ballot(mine >= 0);
    if (any != 0) latest = __shfl(last, 63 - __clzll((long long)any), 64);
    if (found >= 0 && past != 0) {
      drawn = __shfl(mine, __ffsll((unsigned long long)past) - 1, 64);
      break;
    }
    before += __shfl(incl, 63, 64);
  }
  if (lane == 0) a.token[b] = drawn >= 0 ? drawn : latest;
}

}  // namespace

void draft_verify(DType dt, const VerifyArgs& a, hipStream_t s) {
  const int64_t unit = 16 / (int64_t)dtype_size(dt);
  auto whole = [&](const void* p, int64_t row, int64_t slot) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row % unit == 0 && slot % unit == 0;
  };
  const bool wide = whole(a.target, a.t_row, a.t_slot) && (a.draft == nullptr || whole(a.draft, a.d_row, a.d_slot));
  MRT_DTYPE_DISPATCH(dt, {
    if (a.draft != nullptr) hipLaunchKernelGGL((k_verify<T, true>), dim3(a.rows), dim3(64 * kWaves), 0, s, a, wide);
    else hipLaunchKernelGGL((k_verify<T, false>), dim3(a.rows), dim3(64 * kWaves), 0, s, a, wide);
  });
  MRT_HIP_CHECK(hipGetLastError());
}

}  // namespace mrt
