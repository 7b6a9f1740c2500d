// Products in 8-bit integers with a scale for each row (token) and each column (channel):
//   out[m][n] = x_scale[m] w_scale[n] sum_k x[m][k] w[n][k] + add[m][n].
// The sums are whole numbers, exact in 32 bits below k = 2^17 (a term is at most 2^14), so
// how they are cut and ordered changes no bit of a result; a sum is rounded to fp32, and each of
// the two products and the addition by itself, in every kernel.
//
// Few rows (k_i8_few): the weights' bytes bound the product.  A block takes 16 columns, its
// eight waves 128-deep pieces of k in turn; weights go from memory to the matrix cores
// through registers, four lanes to 64 bytes of a row, and one exchange between lanes brings
// them into operand order; the waves' sums meet in LDS.  2 x 1024 by 5632 takes 3.6 us on the
// GPU (1.2 at the rate of a large copy), 16 x 8192 by 8192 21 (14).
//
// Few tiles (k_i8_cut): as above, tiles of 32 x 32, one for each CU at most.
//
// More rows (k_i8_tile): tiles through the LDS ring of ring_gemm.hpp, a k-tile 128 deep, by
// persistent blocks: the k-tiles of all tiles of a block are one stream, so the next tile's
// first k-tiles land while this tile's results are stored.  8192^3 in bf16, a hundred in a row:
// 465 us, 2360 TOP/s, on codes of normal values, 478 on uniform ones (a library's product without
// scales 455 and 453), the matrix cores busy for 67 % of the cycles; 4096^3 67.5.
// 64 x 8192 by 28672, bound by bytes, 54 us, 4.5 TB/s.
#include <algorithm>
#include <type_traits>

#include "codes8.hpp"
#include "i8.hpp"
#include "loose.hpp"
#include "ring_gemm.hpp"

namespace mrt {
namespace {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x16_t __attribute__((ext_vector_type(16)));

// ---- quantisation ------------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ void load16(const T* p, float (&v)[16]) {
  constexpr int kPer = 16 / sizeof(T);
#pragma unroll
  for (int w = 0; w < 16 / kPer; ++w) {
    union {
      uint4 u;
      T x[kPer];
    } r;
    r.u = ld_g16(p + w * kPer);
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[w * kPer + j] = St<T>::ld(r.x[j]);
  }
}

// TH threads a row, 16 values of it each at a time; the first HOLD of a thread's pieces stay
// in registers between the maximum and the codes, longer rows are read again.  Bound by bytes:
// 8192 x 8192 in bf16 takes 32 us, 6.2 TB/s (some of it from the card's last cache).
template <typename T, int TH, int HOLD>
__global__ __launch_bounds__(256) void k_i8_quantize(const T* src, int64_t ld, int rows, int k, int8_t* codes, int64_t ldc,
                                                     float* scales) {
  const int row = blockIdx.x * (256 / TH) + threadIdx.x / TH, at = threadIdx.x % TH, pieces = k / 16;
  const bool there = row < rows;
  const T* from = src + (int64_t)min(row, rows - 1) * ld;
  float v[HOLD][16];
  uint32_t top = 0;
  auto most = [&](const float (&x)[16]) {
#pragma unroll
    for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);  // NaN above all
  };
#pragma unroll
  for (int h = 0; h < HOLD; ++h)
    if (at + h * TH < pieces) {
      load16(from + (at + h * TH) * 16, v[h]);
      most(v[h]);
    }
  for (int p = at + HOLD * TH; p < pieces; p += TH) {
    float x[16];
    load16(from + (int64_t)p * 16, x);
    most(x);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if constexpr (TH > 64) {
    __shared__ uint32_t red[TH / 64];
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TH / 64; ++w) top = max(top, red[w]);
  }
  if (!there) return;
  const float s = codes_scale(top);
  auto put = [&](const float (&x)[16], int p) {
    *reinterpret_cast<uint4*>(codes + (int64_t)row * ldc + (int64_t)p * 16) = codes16(x, s);
  };
#pragma unroll
  for (int h = 0; h < HOLD; ++h)
    if (at + h * TH < pieces) put(v[h], at + h * TH);
  for (int p = at + HOLD * TH; p < pieces; p += TH) {
    float x[16];
    load16(from + (int64_t)p * 16, x);
    put(x, p);
  }
  if (at == 0) scales[row] = s;
}

// ---- few rows ------------------------------------------------------------------------------

constexpr int kWaves = 8;
constexpr int kPiece = 128;  // k of a wave at a time

// Four consecutive results of a row: what goes with their sums, requested before those are
// there.
template <typename T>
struct Four {
  typedef Loose<T, sizeof(T)> Mem;
  union Packed {
    T x[4];
    typename Mem::Word w;
  };
  float by_row, by_col[4];
  Packed old;
  __device__ __forceinline__ void request(const I8Args& a, int row, int col) {
    by_row = ld_g(a.x_scale + min(row, a.rows - 1));
#pragma unroll
    for (int r = 0; r < 4; ++r) by_col[r] = ld_g(a.w_scale + min(col + r, a.n - 1));
    if (a.add == nullptr || row >= a.rows || col >= a.n) return;
    const T* add = static_cast<const T*>(a.add) + row * a.lda + col;
    if (col + 4 <= a.n) {
      old.w = Mem::load(add);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) old.x[r] = add[min(r, a.n - 1 - col)];
    }
  }
  // Scaled and added to step by step, as store_tile does, never in one fused step: which kernel
  // a batch leads to changes no bit of a row.
  __device__ __forceinline__ void store(const I8Args& a, int row, int col, const i32x4_t& sum) {
#pragma clang fp contract(off)
    if (row >= a.rows || col >= a.n) return;
    T* dst = static_cast<T*>(a.out) + row * a.ldo + col;
    Packed u;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float y = (float)sum[r] * by_row * by_col[r];
      u.x[r] = St<T>::st(a.add != nullptr ? y + St<T>::ld(old.x[r]) : y);
    }
    if (col + 4 <= a.n) {
      Mem::store(dst, u.w);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < a.n) dst[r] = u.x[r];
    }
  }
};

template <typename T, int MT>
__global__ __launch_bounds__(64 * kWaves) void k_i8_few(const I8Args a) {
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16;
  const int pieces = (a.k + kPiece - 1) / kPiece;
  __shared__ i32x4_t sums[kWaves][MT][64];
  const int8_t* wrow = a.w + (int64_t)min(n0 + (lane >> 2), a.n - 1) * a.ldw;
  const int8_t* xrow[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) xrow[m] = a.x + (int64_t)min(m * 16 + i, a.rows - 1) * a.ldx;
  struct Piece {
    uint4 w[2], x[MT][2];
  };
  auto load = [&](int p) {
    Piece r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int kw = p * kPiece + h * 64 + (lane & 3) * 16, kx = p * kPiece + h * 64 + g * 16;
      r.w[h] = kw < a.k ? ld_nt16(wrow + kw) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int m = 0; m < MT; ++m) r.x[m][h] = kx < a.k ? ld_g16(xrow[m] + kx) : make_uint4(0, 0, 0, 0);
    }
    return r;
  };
  const int row = wid * 16 + i, col = n0 + g * 4;  // of the results that this wave stores
  Four<T> four;
  if (wid < MT) four.request(a, row, col);
  i32x4_t y[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) y[m] = {0, 0, 0, 0};
  const int pull = (i * 4 + g) * 4;  // the lane with row i's 16 bytes of lane group g
  Piece now = load(wid);
  for (int p = wid; p < pieces; p += kWaves) {
    Piece next = now;
    if (p + kWaves < pieces) next = load(p + kWaves);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint4 u = now.w[h];
      const i32x4_t w = {__builtin_amdgcn_ds_bpermute(pull, u.x), __builtin_amdgcn_ds_bpermute(pull, u.y),
                         __builtin_amdgcn_ds_bpermute(pull, u.z), __builtin_amdgcn_ds_bpermute(pull, u.w)};
#pragma unroll
      for (int m = 0; m < MT; ++m)
        y[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, __builtin_bit_cast(i32x4_t, now.x[m][h]), y[m], 0, 0, 0);
    }
    now = next;
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) sums[wid][m][lane] = y[m];
  __syncthreads();
  if (wid >= MT) return;
  i32x4_t v = sums[0][wid][lane];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) v += sums[w][wid][lane];
  four.store(a, row, col, v);
}

// ---- tiles cut along k -----------------------------------------------------------------------

// Tiles of 32 x 32 whose k eight waves take in turn, 128 at a time, straight from memory: where
// tiles are fewer than CUs, a product takes as long as one tile does, and this one's k-tiles are
// 0.21 us each, those of a 32 x 64 tile through LDS 0.31.  The waves' sums meet in LDS.  More
// pieces on their way (four) or wider tiles (32 x 64) are slower: 33 x 4096 by 4096 10.4 us, 11.2
// and 14.5, through LDS 12.9.
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void k_i8_cut(const I8Args a) {
  constexpr int MT = 2, NT = 2;
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
  const int pieces = (a.k + kPiece - 1) / kPiece;
  __shared__ i32x4_t sums[kWaves][MT * NT][64];
  const int8_t *wrow[NT], *xrow[MT];
#pragma unroll
  for (int n = 0; n < NT; ++n) wrow[n] = a.w + (int64_t)min(n0 + n * 16 + i, a.n - 1) * a.ldw + g * 16;
#pragma unroll
  for (int m = 0; m < MT; ++m) xrow[m] = a.x + (int64_t)min(m0 + m * 16 + i, a.rows - 1) * a.ldx + g * 16;
  struct Piece {
    uint4 w[NT][2], x[MT][2];
  };
  auto load = [&](int p) {
    Piece r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = p * kPiece + h * 64;
      const bool there = k + g * 16 < a.k;
#pragma unroll
      for (int m = 0; m < MT; ++m) r.x[m][h] = there ? ld_g16(xrow[m] + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int n = 0; n < NT; ++n) r.w[n][h] = there ? ld_g16(wrow[n] + k) : make_uint4(0, 0, 0, 0);
    }
    return r;
  };
  static_assert(MT * NT <= kWaves, "a wave stores one tile of 16 x 16");
  const int row = m0 + wid / NT * 16 + i, col = n0 + wid % NT * 16 + g * 4;
  Four<T> four;
  if (wid < MT * NT) four.request(a, row, col);
  i32x4_t y[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) y[m][n] = {0, 0, 0, 0};
  Piece now = load(wid);
  for (int p = wid; p < pieces; p += kWaves) {
    Piece next = now;
    if (p + kWaves < pieces) next = load(p + kWaves);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          y[m][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, now.w[n][h]),
                                                          __builtin_bit_cast(i32x4_t, now.x[m][h]), y[m][n], 0, 0, 0);
    now = next;
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) sums[wid][m * NT + n][lane] = y[m][n];
  __syncthreads();
  i32x4_t v = {0, 0, 0, 0};
  if (wid >= MT * NT) return;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v += sums[w][wid][lane];
  four.store(a, row, col, v);
}

// ---- tiles -----------------------------------------------------------------------------------

// 8-bit operands in the ring: a k-tile is 128 deep, a row of it 8 chunks of 16 bytes.  Chunk c
// of row r is stored at chunk c ^ swz(r), so that 16 consecutive lanes of a fragment read (16
// rows, one chunk) fall in distinct banks.
struct Core8 {
  typedef i32x4_t v8;
  typedef i32x16_t Acc;
  static constexpr int kChunks = 8, kSteps = 4, kParts = 1, kDepth = 128, kProducts = 1;
  static constexpr bool kFine = false;
  __device__ static int swz(int r) { return (r ^ (r >> 3)) & 7; }
  __device__ static int place(int r, int chunk) { return chunk ^ swz(r); }
  __device__ static int chunk_at(int r, int pos) { return pos ^ swz(r); }
  __device__ static int chunk(int step, int, int half) { return 2 * step + half; }
  __device__ __forceinline__ static void mma(const v8 (&a)[1], const v8 (&b)[1], int, i32x16_t& c) {
    c = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[0], a[0], c, 0, 0, 0);
  }
};

__device__ __constant__ uint4 kZeros;  // what k-tiles hold past the end of k

// Results of a wave's tile, whose first row and column are (mb, nb) in the matrix and (mt, nt)
// in the block's tile: a lane holds row mb + 32 i + lane % 32 of tile (i, j) and four times
// four consecutive columns; 16-bit results swap halves between lanes l and l + 32, so that a
// lane stores 16 bytes, and what is added comes the same way, requested kAddAhead tiles ahead
// (in fp32 a second one does not fit the registers).  Rows may begin anywhere: 1000 x 512 by
// 20001 in bf16 takes 36 us, 68 with results stored one by one; by 20000 26.  scale: the block's
// rows' scales, then its columns'.
template <typename T, int BM, int MI, int NJ>
__device__ __forceinline__ void store_tile(const I8Args& a, const i32x16_t (&acc)[MI][NJ], const float* scale, int mb, int nb,
                                           int mt, int nt) {
#pragma clang fp contract(off)
  constexpr bool k16 = sizeof(T) == 2;
  constexpr int kAccesses = k16 ? 2 : 4;  // of 16 bytes, a lane and tile
  constexpr int kAddAhead = k16 ? 2 : 1;
  typedef Loose<T, 4> Mem;
  typedef typename Mem::Word Word;
  const int lane = threadIdx.x & 63, lh = lane >> 5;
  auto column = [&](int h) { return k16 ? 8 * (2 * h + lh) : 8 * h + 4 * lh; };  // of the lane's access h
  const T* add = static_cast<const T*>(a.add);
  Word old[kAddAhead][kAccesses];
  auto request = [&](int x) {  // for tile x % MI, x / MI
    const int row = min(mb + 32 * (x % MI) + (lane & 31), a.rows - 1), first = nb + 32 * (x / MI);
    if (first + 32 > a.n) return;
#pragma unroll
    for (int h = 0; h < kAccesses; ++h) old[x % kAddAhead][h] = Mem::load(add + (int64_t)row * a.lda + first + column(h));
  };
  if (add != nullptr) {
#pragma unroll
    for (int x = 0; x < kAddAhead && x < MI * NJ; ++x) request(x);
  }
#pragma unroll
  for (int x = 0; x < MI * NJ; ++x) {
    const int i = x % MI, j = x / MI;
    const float by_row = scale[mt + 32 * i + (lane & 31)];
    float y[4][4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 v = *reinterpret_cast<const float4*>(scale + BM + nt + 32 * j + 8 * g + 4 * lh);
      const float by_col[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) y[g][r] = (float)acc[i][j][4 * g + r] * by_row * by_col[r];
    }
    const int row = mb + 32 * i + (lane & 31), first = nb + 32 * j;
    const bool there = row < a.rows;
    T* dst = static_cast<T*>(a.out) + (int64_t)row * a.ldo + first;
    if (first + 32 <= a.n) {
      if (add != nullptr) {
#pragma unroll
        for (int h = 0; h < kAccesses; ++h) {
          const Word w = old[x % kAddAhead][h];
          if constexpr (k16) {
            const auto s0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
            const auto s1 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t p[2] = {s0[e], s1[e]};
#pragma unroll
              for (int r = 0; r < 4; ++r) y[2 * h + e][r] += St<T>::unbits((p[r >> 1] >> (16 * (r & 1))) & 0xffffu);
            }
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) y[h][r] += __uint_as_float(w[r]);
          }
        }
        if (x + kAddAhead < MI * NJ) request(x + kAddAhead);
      }
#pragma unroll
      for (int h = 0; h < kAccesses; ++h) {
        Word w;
        if constexpr (k16) {
          auto pack = [&](int g, int r) { return St<T>::bits(y[g][r]) | (St<T>::bits(y[g][r + 1]) << 16); };
          const auto s0 = __builtin_amdgcn_permlane32_swap(pack(2 * h, 0), pack(2 * h + 1, 0), false, false);
          const auto s1 = __builtin_amdgcn_permlane32_swap(pack(2 * h, 2), pack(2 * h + 1, 2), false, false);
          w = {s0[0], s1[0], s0[1], s1[1]};
        } else {
          w = {__float_as_uint(y[h][0]), __float_as_uint(y[h][1]), __float_as_uint(y[h][2]), __float_as_uint(y[h][3])};
        }
        if (there) Mem::store(dst + column(h), w);
      }
    } else {
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int col = 8 * g + 4 * lh + r;
          if (there && first + col < a.n)
            dst[col] = St<T>::st(add != nullptr ? y[g][r] + St<T>::ld(add[(int64_t)row * a.lda + first + col]) : y[g][r]);
        }
    }
  }
}

// Block L takes tiles L, L + gridDim, .. (gridDim % 8 == 0) of the grouped_tile order.  Rows
// and columns past the end are read from the last one and not stored.  TAIL: k is no multiple
// of a k-tile's depth, and what lies past it is read from kZeros.
template <typename T, int BM, int BN, int WM, int WN, int S, bool TAIL>
__global__ __launch_bounds__(64 * WM * WN) void k_i8_tile(const I8Args a) {
  using Core = Core8;
  using Tile = RingTile<Core, BM, BN, WM, WN, S>;
  static_assert(BM + BN <= Tile::kThreads, "a scale a thread");
  extern __shared__ __align__(16) unsigned char lds[];
  __shared__ __attribute__((aligned(16))) float scale[BM + BN];
  const int tid = threadIdx.x, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tm = (a.rows + BM - 1) / BM, tn = (a.n + BN - 1) / BN, tiles = tm * tn;
  const int nk = (a.k + Core::kDepth - 1) / Core::kDepth;
  const int x = blockIdx.x & 7, cnt = (tiles >> 3) + (x < (tiles & 7)), step = gridDim.x >> 3;
  auto origin = [&](int i, int& m0, int& n0) {
    int mt, nt;
    grouped_tile(x + 8 * i, tm, tn, 4, mt, nt);
    m0 = mt * BM;
    n0 = nt * BN;
  };
  int t = blockIdx.x >> 3;
  if (t >= cnt) return;

  // the next k-tile to request: tile lt, depth lk; byte offsets of this thread's chunks from
  // the tile's first rows
  int lt = t, lk = 0;
  const int8_t *ab, *bb;
  uint32_t ao[Tile::LA], bo[Tile::LB];
  auto point = [&]() {
    int m0, n0;
    origin(lt, m0, n0);
    ab = a.x + m0 * a.ldx, bb = a.w + n0 * a.ldw;
#pragma unroll
    for (int q = 0; q < Tile::LA; ++q) {
      int row, chunk;
      Tile::load_pos(q, row, chunk);
      ao[q] = (uint32_t)min(row, a.rows - 1 - m0) * (uint32_t)a.ldx + chunk * 16;
    }
#pragma unroll
    for (int q = 0; q < Tile::LB; ++q) {
      int row, chunk;
      Tile::load_pos(q, row, chunk);
      bo[q] = (uint32_t)min(row, a.n - 1 - n0) * (uint32_t)a.ldw + chunk * 16;
    }
  };
  point();
  auto load = [&](unsigned char* stage) {
    const int8_t *pa = ab + lk * Core::kDepth, *pb = bb + lk * Core::kDepth;
    auto from = [&](const int8_t* p, uint32_t at, int q) {
      if constexpr (!TAIL) return static_cast<const void*>(p + at);
      int row, chunk;
      Tile::load_pos(q, row, chunk);
      return lk * Core::kDepth + chunk * 16 < a.k ? static_cast<const void*>(p + at) : static_cast<const void*>(&kZeros);
    };
#pragma unroll
    for (int q = 0; q < Tile::LA; ++q) Tile::load_a(stage, q, from(pa, ao[q], q));
#pragma unroll
    for (int q = 0; q < Tile::LB; ++q) Tile::load_b(stage, q, from(pb, bo[q], q));
  };
  auto advance = [&] {
    if (++lk == nk) {
      if (lt + step < cnt) {
        lt += step;
        lk = 0;
        point();
      } else {
        lk = nk - 1;  // past the end: the last k-tile again, into a free stage
      }
    }
  };

  typename Tile::State s;
  Tile::start(lds, s, [&](unsigned char* stage) {
    load(stage);
    advance();
  });
  // store instructions of a whole tile's epilogue, 16 bytes each
  constexpr int kStores = Tile::MI * Tile::NJ * (sizeof(T) == 2 ? 2 : 4);
  bool stored = false;  // the previous tile's epilogue issued those, if not more, after the ring's loads
  for (; t < cnt; t += step) {
    int m0, n0;
    origin(t, m0, n0);
    float own = 0.f;  // this thread's scale, which lands while the products run
    if (tid < BM) own = ld_g(a.x_scale + min(m0 + tid, a.rows - 1));
    else if (tid < BM + BN) own = ld_g(a.w_scale + min(n0 + tid - BM, a.n - 1));
    s.clear();
    Tile::reread(lds, s);  // the first fragments need no registers across the epilogue
    for (int kt = 0; kt < nk; ++kt) {
      const bool after = stored && kt == 0;
      Tile::ktile_mixed(lds, s, load, advance, [&] {
        if (after) Tile::template wait_loads<kStores>();
        else Tile::template wait_loads<>();
      });
    }
    if (tid < BM + BN) scale[tid] = own;
    ring_barrier();
    const int mt = (wid / WN) * (BM / WM), nt = (wid % WN) * (BN / WN);
    store_tile<T, BM, Tile::MI, Tile::NJ>(a, s.acc, scale, m0 + mt, n0 + nt, mt, nt);
    asm volatile("" ::: "memory");  // the stores stay ahead of the next tile's waits
    stored = m0 + BM <= a.rows && n0 + BN <= a.n;
  }
  __builtin_amdgcn_s_waitcnt(vm_wait_imm(0));  // no copy into LDS outlives the block
}

template <typename T, int BM, int BN, int WM, int WN, int S>
void launch_tile(const I8Args& a, hipStream_t s) {
  using Tile = RingTile<Core8, BM, BN, WM, WN, S>;
  const int64_t tiles = (int64_t)((a.rows + BM - 1) / BM) * ((a.n + BN - 1) / BN);
  const int64_t grid = std::min<int64_t>(std::max(8, device_cus() & ~7), (tiles + 7) / 8 * 8);
  auto go = [&](auto kernel) {
    allow_dynamic_lds(reinterpret_cast<const void*>(kernel), Tile::kLds);
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(Tile::kThreads), Tile::kLds, s, a);
  };
  if (a.k % Core8::kDepth == 0) go(&k_i8_tile<T, BM, BN, WM, WN, S, false>);
  else go(&k_i8_tile<T, BM, BN, WM, WN, S, true>);
}

template <typename T, int MT>
void launch_few(const I8Args& a, hipStream_t s) {
  hipLaunchKernelGGL((k_i8_few<T, MT>), dim3((a.n + 15) / 16), dim3(64 * kWaves), 0, s, a);
}

// Tiles to choose from, the last, k_i8_cut's, where each has a CU of its own: us that a k-tile
// and the rest of a tile take on a full card (from 4096^3 and 2048 x 1024 by 3200).  Measured and
// chosen (us): 512 x 2816 by 1024 with 256 x 256 / 128 x 128 / 64 x 128 / 32 x 64 tiles 32 / 16.6 /
// 12.0 / 10.0, 2048 x 2816 by 1024 34 / 18.8 / 13.9 / 33, 256 x 4096 by 16384 47 / 25.8 / 31.5 /
// 82, 4096^3 66.8 / 89 / 117 / 318; with 32 x 64 tiles / cut along k 64 x 2816 by 1024 9.7 / 7.3,
// 64 x 8192 by 2048 21.5 / 16.6.
struct TileCost {
  int bm, bn;
  double ktile, rest;
};
constexpr TileCost kTiles[] = {{256, 256, 1.75, 4.0}, {128, 256, 1.13, 2.3}, {128, 128, 0.70, 1.9},
                               {64, 128, 0.45, 1.0},  {32, 128, 0.35, 1.0},  {32, 64, 0.31, 0.8},
                               {32, 32, 0.21, 1.5}};
constexpr int kCut = sizeof(kTiles) / sizeof(kTiles[0]) - 1;

int best_tile(const I8Args& a) {
  const int64_t nk = (a.k + 127) / 128, cus = std::max(8, device_cus() & ~7);
  int best = 0;
  double least = 0.;
  for (int i = 0; i <= kCut; ++i) {
    const TileCost& t = kTiles[i];
    const int64_t tiles = (int64_t)((a.rows + t.bm - 1) / t.bm) * ((a.n + t.bn - 1) / t.bn);
    if (i == kCut && tiles > cus) break;
    const double us = (double)((tiles + cus - 1) / cus) * (nk * t.ktile + t.rest);
    if (i == 0 || us < least) best = i, least = us;
  }
  return best;
}

}  // namespace

void i8_matmul(DType dt, const I8Args& a, hipStream_t s) {
  MRT_DTYPE_DISPATCH(dt, {
    // Few columns give too few tiles to keep the card's loads out, many blocks of k_i8_few read
    // x again (us, k_i8_few / tiles): 2 x 4096 by 4096 7.8 / 12.8, by 16384 19.4 / 14.1; 32 x
    // 4096 by 4096 9.7 / 13.2, by 8192 16.1 / 13.3.
    if (a.rows <= 16 && a.n <= 12288) {
      launch_few<T, 1>(a, s);
    } else if (a.rows <= 32 && a.n <= 6144) {
      launch_few<T, 2>(a, s);
    } else {
      switch (best_tile(a)) {
        case 0: launch_tile<T, 256, 256, 2, 4, 2>(a, s); break;
        case 1: launch_tile<T, 128, 256, 2, 4, 3>(a, s); break;
        case 2: launch_tile<T, 128, 128, 2, 2, 4>(a, s); break;
        case 3: launch_tile<T, 64, 128, 2, 2, 4>(a, s); break;
        case 4: launch_tile<T, 32, 128, 1, 4, 5>(a, s); break;
        case 5: launch_tile<T, 32, 64, 1, 2, 8>(a, s); break;
        default:
          hipLaunchKernelGGL((k_i8_cut<T>), dim3((a.n + 31) / 32, (a.rows + 31) / 32), dim3(64 * kWaves), 0, s, a);
      }
    }
  });
  MRT_HIP_CHECK(hipGetLastError());
}

void i8_quantize(DType dt, const void* src, int64_t ld, int rows, int k, int8_t* codes, int64_t ldc, float* scales,
                 hipStream_t s) {
  MRT_DTYPE_DISPATCH(dt, {
    const T* p = static_cast<const T*>(src);
    if (k <= 1024)
      hipLaunchKernelGGL((k_i8_quantize<T, 64, 1>), dim3((rows + 3) / 4), dim3(256), 0, s, p, ld, rows, k, codes, ldc, scales);
    else if (k <= 4096)
      hipLaunchKernelGGL((k_i8_quantize<T, 256, 1>), dim3(rows), dim3(256), 0, s, p, ld, rows, k, codes, ldc, scales);
    else
      hipLaunchKernelGGL((k_i8_quantize<T, 256, 4>), dim3(rows), dim3(256), 0, s, p, ld, rows, k, codes, ldc, scales);
  });
  MRT_HIP_CHECK(hipGetLastError());
}

}  // namespace mrt
