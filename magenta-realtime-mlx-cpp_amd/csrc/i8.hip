// Products in 8-bit integers with a scale for each row (token) and each column (channel):
//   out[m][n] = x_scale[m] w_scale[n] sum_k x[m][k] w[n][k] + add[m][n].
// The sums are whole numbers, exact in 32 bits below k = 2^17 (a term is at most 2^14), so
// how they are cut and ordered changes no bit of a result.
//
// Few rows (k_i8_few): the weights' bytes bound the product.  A block takes 16 NT columns,
// its eight waves 128-deep pieces of k in turn; weights go from memory to the matrix cores
// through registers, four lanes to 64 bytes of a row, and one exchange between lanes brings
// them into operand order; the waves' sums meet in LDS.
//
// More rows (k_i8_tile): tiles through the LDS ring of ring_gemm.hpp, a k-tile 128 deep, by
// persistent blocks: the k-tiles of all tiles of a block are one stream, so the next tile's
// first k-tiles land while this tile's results are stored.
#include <algorithm>
#include <type_traits>

#include "i8.hpp"
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
// in registers between the maximum and the codes, longer rows are read again.
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
  const float s = top >= 0x7f800000u ? NAN : __uint_as_float(top) * (1.f / 127.f);
  auto put = [&](const float (&x)[16], int p) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float q = s > 0.f ? fminf(fmaxf(rintf(x[4 * j + e] / s), -127.f), 127.f) : 0.f;
        w[j] |= ((uint32_t)(int)q & 0xffu) << (8 * e);
      }
    }
    *reinterpret_cast<uint4*>(codes + (int64_t)row * ldc + (int64_t)p * 16) = make_uint4(w[0], w[1], w[2], w[3]);
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

template <typename T>
__device__ __forceinline__ float result(const I8Args& a, int sum, float by_row, int64_t row, int col) {
  const float y = (float)sum * by_row * a.w_scale[col];
  return a.add != nullptr ? y + St<T>::ld(static_cast<const T*>(a.add)[row * a.lda + col]) : y;
}

template <typename T, int MT, int NT>
__global__ __launch_bounds__(64 * kWaves) void k_i8_few(const I8Args a) {
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
  const int pieces = (a.k + kPiece - 1) / kPiece;
  __shared__ i32x4_t sums[kWaves][NT * MT][64];
  const int8_t* wrow[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) wrow[t] = a.w + (int64_t)min(n0 + t * 16 + (lane >> 2), a.n - 1) * a.ldw;
  const int8_t* xrow[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) xrow[m] = a.x + (int64_t)min(m0 + m * 16 + i, a.rows - 1) * a.ldx;
  struct Piece {
    uint4 w[NT][2], x[MT][2];
  };
  auto load = [&](int p) {
    Piece r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int kw = p * kPiece + h * 64 + (lane & 3) * 16, kx = p * kPiece + h * 64 + g * 16;
#pragma unroll
      for (int t = 0; t < NT; ++t) r.w[t][h] = kw < a.k ? ld_nt16(wrow[t] + kw) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int m = 0; m < MT; ++m) r.x[m][h] = kx < a.k ? ld_g16(xrow[m] + kx) : make_uint4(0, 0, 0, 0);
    }
    return r;
  };
  i32x4_t y[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) y[t][m] = {0, 0, 0, 0};
  const int pull = (i * 4 + g) * 4;  // the lane with row i's 16 bytes of lane group g
  Piece now = load(wid);
  for (int p = wid; p < pieces; p += kWaves) {
    Piece next = now;
    if (p + kWaves < pieces) next = load(p + kWaves);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const uint4 u = now.w[t][h];
        i32x4_t w = {__builtin_amdgcn_ds_bpermute(pull, u.x), __builtin_amdgcn_ds_bpermute(pull, u.y),
                     __builtin_amdgcn_ds_bpermute(pull, u.z), __builtin_amdgcn_ds_bpermute(pull, u.w)};
#pragma unroll
        for (int m = 0; m < MT; ++m)
          y[t][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, __builtin_bit_cast(i32x4_t, now.x[m][h]), y[t][m], 0, 0, 0);
      }
    now = next;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) sums[wid][t * MT + m][lane] = y[t][m];
  __syncthreads();
  for (int z = wid; z < NT * MT; z += kWaves) {
    const int t = z / MT, m = z - t * MT, row = m0 + m * 16 + i, col = n0 + t * 16 + g * 4;
    i32x4_t v = sums[0][z][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += sums[w][z][lane];
    if (row >= a.rows) continue;
    const float by_row = a.x_scale[row];
    T* dst = static_cast<T*>(a.out) + row * a.ldo + col;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (col + r < a.n) dst[r] = St<T>::st(result<T>(a, v[r], by_row, row, col + r));
  }
}

// ---- tiles -----------------------------------------------------------------------------------

// 8-bit operands in the ring: a k-tile is 128 deep, in bytes the same as one of 16-bit
// operands, and so are its places in LDS.
struct Core8 {
  typedef i32x4_t v8;
  typedef i32x16_t Acc;
  static constexpr int kChunks = 8, kSteps = 4, kParts = 1, kDepth = 128, kProducts = 1;
  static constexpr bool kFine = false;
  __device__ static int place(int r, int chunk) { return Core16<bf16>::place(r, chunk); }
  __device__ static int chunk_at(int r, int pos) { return Core16<bf16>::chunk_at(r, pos); }
  __device__ static int chunk(int step, int, int half) { return 2 * step + half; }
  __device__ __forceinline__ static void mma(const v8 (&a)[1], const v8 (&b)[1], int, i32x16_t& c) {
    c = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[0], a[0], c, 0, 0, 0);
  }
};

__device__ __constant__ uint4 kZeros;  // what k-tiles hold past the end of k

// A wave's tile, first row mb, first column nb: a lane holds row mb + 32 i + lane % 32 of
// tile (i, j) and four times four consecutive columns.  wide: rows of out and add take
// vectors of four elements.
template <typename T, int MI, int NJ>
__device__ __forceinline__ void store_tile(const I8Args& a, const i32x16_t (&acc)[MI][NJ], int mb, int nb, bool wide) {
  const int lane = threadIdx.x & 63, lh = lane >> 5;
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = nb + 32 * j + 8 * g + 4 * lh;
      float by_col[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) by_col[r] = a.w_scale[min(col + r, a.n - 1)];
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int row = mb + 32 * i + (lane & 31);
        if (row >= a.rows) continue;
        const float by_row = a.x_scale[row];
        const T* add = static_cast<const T*>(a.add) + row * a.lda + col;
        T* dst = static_cast<T*>(a.out) + row * a.ldo + col;
        union {
          T x[4];
          uint4 w4;
          uint2 w2;
        } u, old;
        const bool whole = wide && col + 4 <= a.n;
        if (a.add != nullptr) {
          if (whole) {
            if constexpr (sizeof(T) == 4) old.w4 = *reinterpret_cast<const uint4*>(add);
            else old.w2 = *reinterpret_cast<const uint2*>(add);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) old.x[r] = col + r < a.n ? add[r] : T(0);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float y = (float)acc[i][j][4 * g + r] * by_row * by_col[r];
          u.x[r] = St<T>::st(a.add != nullptr ? y + St<T>::ld(old.x[r]) : y);
        }
        if (whole) {
          if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst) = u.w4;
          else *reinterpret_cast<uint2*>(dst) = u.w2;
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (col + r < a.n) dst[r] = u.x[r];
        }
      }
    }
}

// Block L takes tiles L, L + gridDim, .. (gridDim % 8 == 0) of the grouped_tile order.  Rows
// and columns past the end are read from the last one and not stored.
template <typename T, int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(64 * WM * WN) void k_i8_tile(const I8Args a, bool wide) {
  using Tile = RingTile<Core8, BM, BN, WM, WN, S>;
  extern __shared__ __align__(16) unsigned char lds[];
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tm = (a.rows + BM - 1) / BM, tn = (a.n + BN - 1) / BN, tiles = tm * tn;
  const int nk = (a.k + Core8::kDepth - 1) / Core8::kDepth;
  const int x = blockIdx.x & 7, cnt = (tiles >> 3) + (x < (tiles & 7)), step = gridDim.x >> 3;
  auto origin = [&](int i, int& m0, int& n0) {
    int mt, nt;
    grouped_tile(x + 8 * i, tm, tn, 4, mt, nt);
    m0 = mt * BM;
    n0 = nt * BN;
  };
  int t = blockIdx.x >> 3;
  if (t >= cnt) return;

  // the next k-tile to request: tile lt, depth lk; this thread's rows in it and chunks
  int lt = t, lk = 0;
  const int8_t *ap[Tile::LA], *bp[Tile::LB];
  int ac[Tile::LA], bc[Tile::LB];
  auto point = [&]() {
    int m0, n0;
    origin(lt, m0, n0);
#pragma unroll
    for (int q = 0; q < Tile::LA; ++q) {
      int row, chunk;
      Tile::load_pos(q, row, chunk);
      ap[q] = a.x + (int64_t)min(m0 + row, a.rows - 1) * a.ldx, ac[q] = chunk * 16;
    }
#pragma unroll
    for (int q = 0; q < Tile::LB; ++q) {
      int row, chunk;
      Tile::load_pos(q, row, chunk);
      bp[q] = a.w + (int64_t)min(n0 + row, a.n - 1) * a.ldw, bc[q] = chunk * 16;
    }
  };
  point();
  auto issue = [&](unsigned char* stage) {
    const int k0 = lk * Core8::kDepth;
    if (k0 + Core8::kDepth <= a.k) {
#pragma unroll
      for (int q = 0; q < Tile::LA; ++q) Tile::load_a(stage, q, ap[q] + k0 + ac[q]);
#pragma unroll
      for (int q = 0; q < Tile::LB; ++q) Tile::load_b(stage, q, bp[q] + k0 + bc[q]);
    } else {
      const int8_t* zero = reinterpret_cast<const int8_t*>(&kZeros);
#pragma unroll
      for (int q = 0; q < Tile::LA; ++q) Tile::load_a(stage, q, k0 + ac[q] < a.k ? ap[q] + k0 + ac[q] : zero);
#pragma unroll
      for (int q = 0; q < Tile::LB; ++q) Tile::load_b(stage, q, k0 + bc[q] < a.k ? bp[q] + k0 + bc[q] : zero);
    }
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
  Tile::start(lds, s, issue);
  for (; t < cnt; t += step) {
    int m0, n0;
    origin(t, m0, n0);
    s.clear();
    Tile::reread(lds, s);  // the first fragments need no registers across the epilogue
    for (int kt = 0; kt < nk; ++kt) Tile::ktile(lds, s, issue, [&] { Tile::template wait_loads<>(); });
    store_tile<T, Tile::MI, Tile::NJ>(a, s.acc, m0 + (wid / WN) * (BM / WM), n0 + (wid % WN) * (BN / WN), wide);
    asm volatile("" ::: "memory");  // the stores stay ahead of the next tile's waits
  }
  __builtin_amdgcn_s_waitcnt(vm_wait_imm(0));  // no copy into LDS outlives the block
}

template <typename T, int BM, int BN, int WM, int WN, int S>
void launch_tile(const I8Args& a, bool wide, hipStream_t s) {
  using Tile = RingTile<Core8, BM, BN, WM, WN, S>;
  const auto kernel = &k_i8_tile<T, BM, BN, WM, WN, S>;
  allow_dynamic_lds(reinterpret_cast<const void*>(kernel), Tile::kLds);
  const int64_t tiles = (int64_t)((a.rows + BM - 1) / BM) * ((a.n + BN - 1) / BN);
  const int64_t grid = std::min<int64_t>(std::max(8, device_cus() & ~7), (tiles + 7) / 8 * 8);
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(Tile::kThreads), Tile::kLds, s, a, wide);
}

template <typename T, int MT>
void launch_few(const I8Args& a, hipStream_t s) {
  const int tiles = (a.n + 15) / 16;
  const dim3 grid((tiles + 1) / 2, (a.rows + 16 * MT - 1) / (16 * MT));
  if (tiles < 1024) hipLaunchKernelGGL((k_i8_few<T, MT, 1>), dim3(tiles, grid.y), dim3(64 * kWaves), 0, s, a);
  else hipLaunchKernelGGL((k_i8_few<T, MT, 2>), grid, dim3(64 * kWaves), 0, s, a);
}

}  // namespace

void i8_matmul(DType dt, const I8Args& a, hipStream_t s) {
  MRT_DTYPE_DISPATCH(dt, {
    const size_t unit = 4 * sizeof(T);
    const bool wide = reinterpret_cast<uintptr_t>(a.out) % unit == 0 && a.ldo % 4 == 0 &&
                      (a.add == nullptr || (reinterpret_cast<uintptr_t>(a.add) % unit == 0 && a.lda % 4 == 0));
    if (a.rows <= 16) launch_few<T, 1>(a, s);
    else if (a.rows <= 32) launch_few<T, 2>(a, s);
    else if (a.rows <= 64) launch_few<T, 4>(a, s);
    else {
      const int64_t big = (int64_t)((a.rows + 255) / 256) * ((a.n + 255) / 256);
      const int64_t mid = (int64_t)((a.rows + 127) / 128) * ((a.n + 127) / 128);
      if (big >= 192) launch_tile<T, 256, 256, 2, 4, 2>(a, wide, s);
      else if (mid >= 192) launch_tile<T, 128, 128, 2, 2, 4>(a, wide, s);
      else launch_tile<T, 64, 64, 2, 2, 6>(a, wide, s);
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
