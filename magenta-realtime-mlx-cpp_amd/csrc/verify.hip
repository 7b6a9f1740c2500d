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
// Each node's own p(x) and q(x) are gathered at once, so tests need no memory; a rejection
// costs one pass over the slot's rows.  Sums are taken by segments of the vocabulary, a wave
// each, and the drawn token's segment is the only one looked at again.  k_verify does all of
// it, a block a sequence.  What bounds that is one CU's share of arithmetic in 64 bits, so over
// large vocabularies the first passes are made by many blocks, a launch each (k_verify_pass):
// every block takes the walk up where the launch before stopped, goes on by that one's sums as
// far as they reach, which takes no memory, and sums its segments of the pass that is needed
// next.  Passes beyond those launches are k_verify's own.  Sums are the same either way, bit
// for bit.  Bound by launches then, which follow each other: 16 trees of 31 nodes over 131072
// tokens in fp32 take 38 us in seven of them for 17 MB that they have to read (4 us at the rate
// of a large copy); a chain of 16 nodes over 1024 tokens is one of 6 us, and 9 from Python.
#include <algorithm>
#include <type_traits>

#include "device_utils.hpp"
#include "loose.hpp"
#include "verify.hpp"

namespace mrt {
namespace {

constexpr int kWaves = 16;
constexpr int kSegments = 256;
constexpr int kAhead = 4;  // loads of a wave that are on their way: a pass by one block 43 us with one, 35 with four
// Vocabulary from which passes are made by many blocks.  32 chains of 16, drawn (us, one block /
// many): 16000 in fp32 11.6 / 12.4, 29824 in fp32 15.6 / 12.6, in bf16 13.7 / 12.8; 16 of 131072
// in fp32 32.9 / 13.2.
constexpr int kManyVocab = 24000;
// Launches of passes for trees, of 31 nodes with 1.6 passes on average; the most among 16
// sequences is three to six, a launch that nobody needs takes 2 to 3 us, a pass by one block 35.
// 16 x 131072 with 0 / 5 / 7 / 9: 152 / 43 / 42 / 45 us, 2 x 131072 with 4 / 6: 21 / 25.
constexpr int tree_rounds(int rows) { return rows <= 4 ? 4 : 6; }

// What is not a positive finite number counts as 0.
__device__ __forceinline__ float counted(float p) {
  return __builtin_amdgcn_classf(p, 0x180) ? p : 0.f;  // positive, normal or not
}

// VEC consecutive probabilities; 0 past the end.  Rows may begin anywhere.
template <typename T, int VEC>
__device__ __forceinline__ uint4 load_raw(const T* row, int at, int V) {
  union {
    T x[VEC];
    uint4 w;
    typename Loose<T, 4>::Word v;
  } u;
  if (at + VEC <= V) {
    u.v = Loose<T, 4>::load(row + at);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) u.x[e] = at + e < V ? ld_g(row + at + e) : T(0);
  }
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

__device__ __forceinline__ double lane_of(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)u, lane), hi = __builtin_amdgcn_readlane((uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float lane_of(float v, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}
__device__ __forceinline__ int lane_of(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// The rejections at a slot, the k-th in lane k of every wave: Z before it, the token.
struct Rejections {
  double z;
  int token;
};

// r of element `at` after n rejections, at most M of them in registers (absent ones change
// nothing); M -1: any number.
template <bool DRAFT, int M>
struct Rest {
  double z[M > 0 ? M : 1];
  int token[M > 0 ? M : 1];
  const Rejections& rej;
  int n;
  __device__ __forceinline__ Rest(const Rejections& r, int n_) : rej(r), n(n_) {
#pragma unroll
    for (int k = 0; k < M; ++k) z[k] = k < n ? lane_of(rej.z, k) : 0.0, token[k] = k < n ? lane_of(rej.token, k) : -1;
  }
  __device__ __forceinline__ double operator()(float p, float q, int at) const {
    double r = (double)p;
    auto fold = [&](double zk, int tk) {
      if constexpr (DRAFT) r = fmax(fma(-zk, (double)q, r), 0.0);
      else r = at == tk ? 0.0 : r;
    };
    if constexpr (M < 0) {
      for (int k = 0; k < n; ++k) fold(lane_of(rej.z, k), lane_of(rej.token, k));
    } else {
#pragma unroll
      for (int k = 0; k < M; ++k) fold(z[k], token[k]);
    }
    return r;
  }
};

// A sequence's nodes, node t in lane t of every wave.
struct Nodes {
  int parent, token;  // -2, -1: not there
  float p, q, u;      // of its token at its slot, its random number
};

// Sums over a slot, by segments, in LDS.
struct Sums {
  double seg[kSegments];  // running over the segments
  double total;
};

// How the vocabulary is cut: chunks of 64 lanes, `per` of them a segment.
template <typename T>
struct Cut {
  static constexpr int VEC = 16 / sizeof(T), CHUNK = 64 * VEC;
  int chunks, per, segments;
  __host__ __device__ explicit Cut(int V)
      : chunks((V + CHUNK - 1) / CHUNK), per((chunks + kSegments - 1) / kSegments), segments((chunks + per - 1) / per) {}
};

template <typename T, bool DRAFT>
__device__ __forceinline__ Nodes gather(const VerifyArgs& a, int b, int lane) {
  const int N = a.nodes, t = min(lane, N - 1);
  const T* target = static_cast<const T*>(a.target) + b * a.t_row;
  const T* draft = static_cast<const T*>(a.draft) + b * a.d_row;
  const int up = a.parents != nullptr ? a.parents[b * a.parents_stride + t] : t - 1;
  const int x = a.tokens[(int64_t)b * N + t];
  Nodes s;
  s.u = a.uniforms[(int64_t)b * (N + 1) + t];
  const bool there = lane < N && up >= -1 && up < t, known = x >= 0 && x < a.vocab;
  s.parent = there ? up : -2;
  s.token = known ? x : -1;
  const int slot = there ? up + 1 : 0, at = known ? x : 0;
  s.p = counted(St<T>::ld(ld_g(target + slot * a.t_slot + at)));
  s.q = DRAFT ? counted(St<T>::ld(ld_g(draft + slot * a.d_slot + at))) : 1.f;
  return s;
}

// Sums of r after n rejections at slot `at`, of the segments first, first + W, .. below
// `last`, by W waves: put(segment, sum).
template <typename T, bool DRAFT, int W, int M, class Put>
__device__ __forceinline__ void sum_segments_of(const VerifyArgs& a, const Cut<T>& cut, int b, int at, int n,
                                                const Rejections& rej, int first, int last, Put&& put) {
  constexpr int VEC = Cut<T>::VEC, CHUNK = Cut<T>::CHUNK;
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T* p = static_cast<const T*>(a.target) + b * a.t_row + at * a.t_slot;
  const T* q = static_cast<const T*>(a.draft) + b * a.d_row + at * a.d_slot;
  constexpr bool both = DRAFT && M != 0;
  const Rest<DRAFT, M> r(rej, n);
  // A wave's chunks, kAhead of them on their way.
  const int from = first + wid, mine = from < last ? ((last - 1 - from) / W + 1) * cut.per : 0;
  auto chunk_of = [&](int k) { return (from + k / cut.per * W) * cut.per + k % cut.per; };
  uint4 pr[kAhead], qr[kAhead];
  auto load = [&](int k, int j) {
    const int x = chunk_of(min(k, mine - 1)) * CHUNK + lane * VEC;
    pr[j] = load_raw<T, VEC>(p, x, a.vocab);
    if constexpr (both) qr[j] = load_raw<T, VEC>(q, x, a.vocab);
  };
  if (mine > 0) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) load(j, j);
  }
  double sum = 0.0;
  for (int k0 = 0; k0 < mine; k0 += kAhead) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int k = k0 + j;
      if (k >= mine) break;
      const int x = chunk_of(k) * CHUNK + lane * VEC;
      float pv[VEC], qv[VEC] = {};
      unpack<T, VEC>(pr[j], pv);
      if constexpr (both) unpack<T, VEC>(qr[j], qv);
      if (k + kAhead < mine) load(k + kAhead, j);
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum += r(pv[e], qv[e], x + e);
      if ((k + 1) % cut.per == 0) {
        sum = wave_sum(sum);
        if (lane == 0) put(from + k / cut.per * W, sum);
        sum = 0.0;
      }
    }
  }
}

template <typename T, bool DRAFT, int W, class Put>
__device__ __forceinline__ void sum_segments(const VerifyArgs& a, const Cut<T>& cut, int b, int at, int n,
                                             const Rejections& rej, int first, int last, Put&& put) {
  if (n == 0) sum_segments_of<T, DRAFT, W, 0>(a, cut, b, at, n, rej, first, last, put);
  else if (n <= 2) sum_segments_of<T, DRAFT, W, 2>(a, cut, b, at, n, rej, first, last, put);
  else sum_segments_of<T, DRAFT, W, -1>(a, cut, b, at, n, rej, first, last, put);
}

// s.seg from the segments' sums to running ones, and s.total; by the whole block.  Running
// sums never fall, a segment without weight adds nothing to them, and the last one is the total,
// whatever the roundings: at each level of the scan the right half's lanes add the left half's
// last sum to their own, and a lane's last segment takes the lane's sum itself.  So the first
// that exceeds a threshold is of a segment with weight, and none exceeds the total.
__device__ __forceinline__ void run_sums(Sums& s, int segments) {
  const int lane = threadIdx.x & 63;
  __syncthreads();
  if (threadIdx.x < 64) {  // four segments a lane
    double v[4], run = 0.0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      run += lane * 4 + k < segments ? s.seg[lane * 4 + k] : 0.0;
      v[k] = run;
    }
    double incl = run;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl(incl, (lane & -o) - 1, 64);  // of the right half's lanes: the left half's last
      if (lane & o) incl += y;
    }
    double before = __shfl_up(incl, 1, 64);
    if (lane == 0) before = 0.0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (lane * 4 + k < segments) s.seg[lane * 4 + k] = v[k] == run ? incl : fmin(before + v[k], incl);
    if (lane == 63) s.total = incl;
  }
  __syncthreads();
}

// The walk, the same in every wave of a sequence's blocks: it stops where it needs the sums of a
// pass, and goes on from there, in the same launch or the next.
struct Walk {
  enum { kTest = -1, kLast = -2, kBare = -3 };
  int here, n, count;  // the slot, rejections there, nodes accepted
  int wait;            // what the sums are for: the test of a node (its id), the last draw, that from the target itself
  uint64_t kids;       // children of `here` that are left
  double z;
  int path;            // lane k: the k-th accepted node
  Rejections rej;

  // The children of a node, in order; nothing was drawn for what is not a token.
  __device__ __forceinline__ static uint64_t children(const Nodes& node, int parent) {
    return __ballot(node.parent == parent && node.token >= 0);
  }
  __device__ __forceinline__ void begin(const Nodes& node) {
    here = n = count = 0, wait = kTest, z = 1.0, path = -1, rej = {0.0, -1};
    kids = children(node, -1);
  }
  // Goes on, with the sum of the pass that it stopped for.  True: the walk has ended, and the
  // last sums are those of its draw; else it needs those of r at slot `here` after n rejections.
  template <bool DRAFT>
  __device__ __forceinline__ bool go(const Nodes& node, int lane, double total) {
    if (wait == kBare) return true;
    if (wait == kLast) {
      if (total > 0.0 || n == 0) return true;
      n = 0, wait = kBare;  // nothing left: the target itself
      return false;
    }
    if (wait >= 0) z = total;
    for (;;) {
      int t = wait;
      wait = kTest;
      if (t < 0) {
        if (kids == 0) {
          wait = kLast;
          return false;
        }
        t = __ffsll((unsigned long long)kids) - 1;
        kids &= kids - 1;
        if (DRAFT && n > 0) {
          wait = t;
          return false;
        }
      }
      const int x = lane_of(node.token, t);
      const float q = lane_of(node.q, t);
      const double r = Rest<DRAFT, -1>(rej, n)(lane_of(node.p, t), q, x);
      if ((double)lane_of(node.u, t) * z * (double)q < r) {
        path = lane == count ? t : path;
        ++count;
        here = t + 1, n = 0, z = 1.0;
        kids = children(node, t);
      } else {
        rej.z = lane == n ? z : rej.z, rej.token = lane == n ? x : rej.token;
        if (!DRAFT) z -= r;
        ++n;
      }
    }
  }
};

// A walk between two launches, and its nodes.
struct Saved {
  double z, rej_z[64];
  uint64_t kids;
  int here, n, count, wait;
  int rej_token[64], path[64], parent[64], token[64];
  float p[64], q[64], u[64];

  __device__ __forceinline__ void put(const Walk& w, const Nodes& x, int lane) {
    rej_z[lane] = w.rej.z, rej_token[lane] = w.rej.token, path[lane] = w.path;
    parent[lane] = x.parent, token[lane] = x.token, p[lane] = x.p, q[lane] = x.q, u[lane] = x.u;
    if (lane == 0) z = w.z, kids = w.kids, here = w.here, n = w.n, count = w.count, wait = w.wait;
  }
  __device__ __forceinline__ void get(Walk& w, Nodes& x, int lane) const {
    w.rej = {ld_g(rej_z + lane), ld_g(rej_token + lane)}, w.path = ld_g(path + lane);
    x.parent = ld_g(parent + lane), x.token = ld_g(token + lane), x.p = ld_g(p + lane), x.q = ld_g(q + lane);
    x.u = ld_g(u + lane);
    const double z0 = ld_g(&z);
    const uint64_t k0 = ld_g(&kids);
    const int h0 = ld_g(&here), n0 = ld_g(&n), c0 = ld_g(&count), w0 = ld_g(&wait);
    w.z = lane_of(z0, 0);
    w.kids = (uint64_t)(uint32_t)lane_of((int)(k0 >> 32), 0) << 32 | (uint32_t)lane_of((int)k0, 0);
    w.here = lane_of(h0, 0), w.n = lane_of(n0, 0), w.count = lane_of(c0, 0), w.wait = lane_of(w0, 0);
  }
};

// What goes from launch to launch.  A launch reads what the one before wrote and writes the
// other of two halves; the walk and sums of a sequence whose walk has ended stay.
struct Between {
  Saved* saved;  // (2, rows)
  double* sums;  // (2, rows, kSegments)
  int* ended;    // (2, rows) 0, or the launch that found it ended
  static size_t bytes(int rows) { return (size_t)rows * (2 * sizeof(Saved) + 2 * kSegments * 8 + 8); }
  Between(void* ws, int rows)
      : saved(static_cast<Saved*>(ws)),
        sums(reinterpret_cast<double*>(saved + 2 * (size_t)rows)),
        ended(reinterpret_cast<int*>(sums + 2 * (size_t)rows * kSegments)) {}
  __device__ __forceinline__ Saved& walk_of(int launch, int rows, int b) const { return saved[(int64_t)(launch & 1) * rows + b]; }
  __device__ __forceinline__ int& ended_of(int launch, int rows, int b) const { return ended[(int64_t)(launch & 1) * rows + b]; }
  __device__ __forceinline__ double* sums_of(int launch, int rows, int b) const {
    return sums + ((int64_t)(launch & 1) * rows + b) * kSegments;
  }
};

// Launch `round` of passes: block (x, b) sums segments x share .. of sequence b.
template <typename T, bool DRAFT>
__global__ __launch_bounds__(256) void k_verify_pass(const VerifyArgs a, int round, int share, const Between mem) {
  const Cut<T> cut(a.vocab);
  const int b = blockIdx.y, first = blockIdx.x * share, last = min(first + share, cut.segments);
  const int tid = threadIdx.x, lane = tid & 63;
  __shared__ Sums s;
  Nodes node;
  Walk walk;
  bool ended = false;
  if (round == 0) {
    node = gather<T, DRAFT>(a, b, lane);
    walk.begin(node);
    walk.go<DRAFT>(node, lane, 0.0);
  } else {
    const int over = ld_g(&mem.ended_of(round - 1, a.rows, b));
    if (over != 0) {
      if (blockIdx.x == 0 && tid == 0) mem.ended_of(round, a.rows, b) = over;
      return;
    }
    if (tid < cut.segments) s.seg[tid] = ld_g(mem.sums_of(round - 1, a.rows, b) + tid);
    mem.walk_of(round - 1, a.rows, b).get(walk, node, lane);
    run_sums(s, cut.segments);
    ended = walk.go<DRAFT>(node, lane, s.total);
  }
  if (blockIdx.x == 0 && tid < 64) {
    mem.walk_of(round, a.rows, b).put(walk, node, lane);
    if (lane == 0) mem.ended_of(round, a.rows, b) = ended ? round : 0;
  }
  if (ended) return;
  double* to = mem.sums_of(round, a.rows, b);
  sum_segments<T, DRAFT, 4>(a, cut, b, walk.here, walk.n, walk.rej, first, last, [&](int x, double v) { to[x] = v; });
}

// The rest, a block a sequence, after `rounds` launches of passes.
template <typename T, bool DRAFT>
__global__ __launch_bounds__(64 * kWaves) void k_verify(const VerifyArgs a, int rounds, const Between mem) {
  constexpr int VEC = Cut<T>::VEC, CHUNK = Cut<T>::CHUNK;
  const Cut<T> cut(a.vocab);
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int N = a.nodes, V = a.vocab, per = cut.per, chunks = cut.chunks, segments = cut.segments;
  __shared__ Sums s;
  Nodes node;
  Walk walk;
  bool ended = false;
  if (rounds == 0) {
    node = gather<T, DRAFT>(a, b, lane);
    walk.begin(node);
    walk.go<DRAFT>(node, lane, 0.0);
  } else {
    const int at = __builtin_amdgcn_readfirstlane(ld_g(&mem.ended_of(rounds - 1, a.rows, b)));
    if (tid < segments) s.seg[tid] = ld_g(mem.sums_of(at != 0 ? at - 1 : rounds - 1, a.rows, b) + tid);
    mem.walk_of(at != 0 ? at : rounds - 1, a.rows, b).get(walk, node, lane);
    run_sums(s, segments);
    ended = at != 0 || walk.go<DRAFT>(node, lane, s.total);
  }
  while (!ended) {
    __syncthreads();  // the pass before has been read
    sum_segments<T, DRAFT, kWaves>(a, cut, b, walk.here, walk.n, walk.rej, 0, segments, [&](int x, double v) { s.seg[x] = v; });
    run_sums(s, segments);
    ended = walk.go<DRAFT>(node, lane, s.total);
  }
  const int here = walk.here, n = walk.n;
  const Rest<DRAFT, -1> rest(walk.rej, n);
  if (tid < N) a.accepted[(int64_t)b * N + tid] = tid < walk.count ? walk.path : -1;
  if (tid == 0) a.count[b] = walk.count;
  if (wid != 0) return;

  // The first segment that exceeds the threshold, then its first chunk, lane, token.
  const double sum = s.total, want = fmax(a.uniforms[(int64_t)b * (N + 1) + N] * sum, 0.0);
  int found = -1;
  for (int s0 = 0; s0 < segments && found < 0; s0 += 64) {
    const uint64_t past = __ballot(s0 + lane < segments && s.seg[s0 + lane] > want);
    if (past != 0) found = s0 + __ffsll((unsigned long long)past) - 1;
  }
  int drawn = -1, latest = -1;  // latest: the last token with a positive r seen
  const T* p = static_cast<const T*>(a.target) + b * a.t_row + here * a.t_slot;
  const T* q = static_cast<const T*>(a.draft) + b * a.d_row + here * a.d_slot;
  const bool both = DRAFT && n > 0;
  // Without one (a random number of 1): the last token with any weight, over all segments.
  int c = found < 0 ? 0 : found * per;
  const int end = found < 0 ? chunks : min((found + 1) * per, chunks);
  double before = found > 0 ? s.seg[found - 1] : 0.0;
  for (; c < end && sum > 0.0; ++c) {
    const int at = c * CHUNK + lane * VEC;
    float pv[VEC], qv[VEC];
    unpack<T, VEC>(load_raw<T, VEC>(p, at, V), pv);
    if (both) unpack<T, VEC>(load_raw<T, VEC>(q, at, V), qv);
    double v[VEC], run = 0.0;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      v[e] = rest(pv[e], both ? qv[e] : 0.f, at + e);
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

// Passes made by many blocks, a launch each.
int rounds_of(const VerifyArgs& a) {
  if (a.vocab < kManyVocab || a.rows >= 256) return 0;
  return a.draft == nullptr || a.parents == nullptr ? 1 : tree_rounds(a.rows);  // a chain has one, as have drafts that were not drawn
}

}  // namespace

size_t draft_verify_workspace(const VerifyArgs& a) { return rounds_of(a) > 0 ? Between::bytes(a.rows) : 0; }

void draft_verify(DType dt, const VerifyArgs& a, void* ws, hipStream_t s) {
  const int rounds = rounds_of(a);
  const Between mem(ws, a.rows);
  MRT_DTYPE_DISPATCH(dt, {
    auto go = [&](auto drawn) {
      constexpr bool DRAFT = decltype(drawn)::value;
      const Cut<T> cut(a.vocab);
      // four segments a block, a wave each, or as many as give the card two blocks a CU
      const int blocks = std::max(1, std::min((cut.segments + 3) / 4, 512 / a.rows));
      const int share = (cut.segments + blocks - 1) / blocks;
      const dim3 grid((cut.segments + share - 1) / share, a.rows);
      for (int r = 0; r < rounds; ++r)
        hipLaunchKernelGGL((k_verify_pass<T, DRAFT>), grid, dim3(256), 0, s, a, r, share, mem);
      hipLaunchKernelGGL((k_verify<T, DRAFT>), dim3(a.rows), dim3(64 * kWaves), 0, s, a, rounds, mem);
    };
    if (a.draft != nullptr) go(std::true_type{});
    else go(std::false_type{});
  });
  MRT_HIP_CHECK(hipGetLastError());
}

}  // namespace mrt
