// MXFP4 (mx4.h): quantisation along rows and columns, the values back, and the
// product of two quantised matrices (gfx950).
//
//  * mx_quantize: codes and scales of a matrix, of its transpose, or of both
//    from one read.  Bound by the bytes it reads and writes.
//  * mx_dequantize: the values that codes and scales stand for.
//  * mx_gemm: C = A B^T over the values, v_mfma_scale_f32_*_f8f6f4 with fp4
//    operands (the matrix cores multiply by the two blocks' scales), sums in
//    fp32, one rounding at the end.
#include <type_traits>

#include "mx4.h"

namespace sfp8 {

// ---------------------------------------------------------------------------
// Quantisation
// ---------------------------------------------------------------------------
SFP8_DEV uint32_t max_u(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int CTRL>
SFP8_DEV uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true);
}

struct MxQuantArgs {
  const void* x;
  int64_t R, C, ld, batch_stride;  // elements
  uint8_t *codes, *scales;         // of x, or NULL
  uint8_t *codes_t, *scales_t;     // of its transpose, or NULL
};

// One work-group takes ITER times 2048 values in rows of WIDE.  WIDE / 8 lanes hold
// those of a row (four lanes a block: its maximum is two lane exchanges away), so
// the row codes leave straight from the registers, four rows of 64 bytes in one run.
// For the columns the values pass through LDS as they are: a lane then holds
// 32 values of one column (16-bit types in the wide tile: of two), so neither its
// maximum nor its codes need another lane; the codes go back through LDS so that
// each column's 64 bytes and the tile's 8 KiB are written in one run.
// 128 x 128 values where there are columns, half as wide where those tiles would
// leave CUs without one; along rows alone 32 x 128 there.
template <int DT, bool ROWS, bool COLS, int ITER, int WIDE>
__global__ __launch_bounds__(256) void mx_quantize_kernel(MxQuantArgs a) {
  constexpr int kSize = DT == kMxF32 ? 4 : 2, kLanes = WIDE / 8, kRows = 256 / kLanes, kTall = kRows * ITER;
  static_assert(kTall == 128 || !COLS, "a slab of the transpose");
  __shared__ __align__(16) uint8_t raw[COLS ? 128 * WIDE * kSize : 16];
  __shared__ __align__(16) uint8_t out[COLS ? WIDE * 64 : 16];
  __shared__ __align__(16) uint8_t out_scale[COLS ? WIDE * 4 : 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t slabs = mx_slabs(a.C), nx = slabs * (128 / WIDE), ny = (a.R + kTall - 1) / kTall;
  const int64_t id = blockIdx.x, cs = id % nx, rs = id / nx % ny, z = id / nx / ny;
  const int64_t c0 = cs * WIDE, r0 = rs * kTall, rows = mx_rows(a.R), cols = mx_rows(a.C);
  const uint8_t* x = reinterpret_cast<const uint8_t*>(a.x) + z * a.batch_stride * kSize;
  const int col = 8 * (tid % kLanes), sub = tid / kLanes;

  Eight<DT> v[ITER];
  if (c0 + WIDE <= a.C && r0 + kTall <= a.R) {
#pragma unroll
    for (int i = 0; i < ITER; ++i) v[i] = load8<DT>(x, (r0 + kRows * i + sub) * a.ld + c0 + col);
  } else {
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int64_t r = r0 + kRows * i + sub;
      v[i] = Eight<DT>{};
      if (r < a.R && c0 + col < a.C) v[i] = load8_upto<DT>(x, r * a.ld + c0 + col, a.C - c0 - col);
    }
  }
  if constexpr (ROWS) {
    const int64_t slab = z * slabs + cs / (128 / WIDE);
    const int in = (int)(cs % (128 / WIDE)) * WIDE;  // the tile's first column in its slab
    uint8_t* codes = a.codes + slab * rows * 64 + in / 2;
    uint8_t* scales = a.scales + slab * rows * 4 + in / 32;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      uint32_t m = abs_max8<DT>(v[i]);
      m = max_u(m, dpp<0xB1>(m));
      m = max_u(m, dpp<0x4E>(m));
      const uint32_t e = mx_scale_code(abs_bits_to_f32<DT>(m));
      const uint32_t c = codes8<DT>(v[i], mx_scale_value(e));
      uint32_t s = e << (8 * (tid % kLanes / 4));  // the row's four scales (or two) in one word
      s |= dpp<0x141>(s);
      if constexpr (WIDE == 128) s |= dpp<0x140>(s);
      const int64_t r = r0 + kRows * i + sub;
      if (r < rows) {
        *reinterpret_cast<uint32_t*>(codes + r * 64 + col / 2) = c;
        if (col == 0) {
          if constexpr (WIDE == 128) *reinterpret_cast<uint32_t*>(scales + r * 4) = s;
          else *reinterpret_cast<uint16_t*>(scales + r * 4) = (uint16_t)s;
        }
      }
    }
  }
  if constexpr (COLS) {
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      uint32_t* p = reinterpret_cast<uint32_t*>(raw + ((kRows * i + sub) * WIDE + col) * kSize);
      *reinterpret_cast<intx4*>(p) = intx4{(int)v[i].w[0], (int)v[i].w[1], (int)v[i].w[2], (int)v[i].w[3]};
      if constexpr (DT == kMxF32)
        *reinterpret_cast<intx4*>(p + 4) = intx4{(int)v[i].w[4], (int)v[i].w[5], (int)v[i].w[6], (int)v[i].w[7]};
    }
    __syncthreads();
    // 64 columns of the wave's 32 rows a turn, one a lane; or 128 where a lane's word holds two
    constexpr int kWords = WIDE * kSize / 4, kCols = kWords * 2 == WIDE && WIDE == 128 ? 2 : 1;
#pragma unroll
    for (int h = 0; h < WIDE / 64 / kCols; ++h) {
      const int first = 64 * h + kCols * lane;  // this lane's column
      const uint32_t* p = reinterpret_cast<const uint32_t*>(raw) + 32 * wave * kWords + first * kSize / 4;
      uint32_t w[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) w[i] = p[i * kWords];
#pragma unroll
      for (int half = 0; half < kCols; ++half) {
        const int k = kCols == 2 ? half : first & 1;  // the column's half of the word
        Eight<DT> q[4];
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (DT == kMxF32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[j].w[i] = w[8 * j + i];
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t lo = w[8 * j + 2 * i], hi = w[8 * j + 2 * i + 1];
              q[j].w[i] = k ? (lo >> 16) | (hi & 0xffff0000u) : (lo & 0xffffu) | (hi << 16);
            }
          }
          m = max_u(m, abs_max8<DT>(q[j]));
        }
        const uint32_t e = mx_scale_code(abs_bits_to_f32<DT>(m));
        const float s = mx_scale_value(e);
        const int c = first + half;
        // 16-byte chunk `wave` of column c, at chunk wave ^ (c / 2) % 4: the lanes of a store spread over the banks
        *reinterpret_cast<intx4*>(out + c * 64 + 16 * (wave ^ ((c >> 1) & 3))) =
            intx4{(int)codes8<DT>(q[0], s), (int)codes8<DT>(q[1], s), (int)codes8<DT>(q[2], s),
                  (int)codes8<DT>(q[3], s)};
        out_scale[c * 4 + wave] = (uint8_t)e;
      }
    }
    __syncthreads();
    uint8_t* codes = a.codes_t + (z * ny + rs) * cols * 64;
    uint8_t* scales = a.scales_t + (z * ny + rs) * cols * 4;
#pragma unroll
    for (int j = 0; j < WIDE / 64; ++j) {
      const int u = tid + 256 * j, c = u >> 2, ch = u & 3;
      if (c0 + c < cols)
        *reinterpret_cast<intx4*>(codes + (c0 + c) * 64 + 16 * ch) =
            *reinterpret_cast<const intx4*>(out + c * 64 + 16 * (ch ^ ((c >> 1) & 3)));
    }
    if (tid < WIDE && c0 + tid < cols)
      *reinterpret_cast<uint32_t*>(scales + (c0 + tid) * 4) = reinterpret_cast<const uint32_t*>(out_scale)[tid];
  }
}

// Work-groups for tiles of 128 x 128 and, where those would not be two for each
// CU, of 32 x 128 along rows (5003 x 1001: 4.2 us against 5.2; 65536 x 1024 27.9
// against 26.1); where they would not be one, of 128 x 64 along columns (rows and
// columns of 1030 x 1000 in fp32 4.1 against 5.4, of 2003 x 1030 in bf16 6.1 against
// 7.5; of 4096 x 1024 in bf16 5.4 against 5.1).  One limit for all types: fp32 tiles
// of 128 x 128 have 74 KB of LDS, two a CU, and were not timed against narrow ones past it.
struct MxGrid {
  unsigned tall, low;
  MxGrid(int64_t batch, int64_t R, int64_t C)
      : tall((unsigned)(batch * mx_slabs(C) * ((R + 127) / 128))),
        low(tall >= 512 ? 0 : (unsigned)(batch * mx_slabs(C) * ((R + 31) / 32))) {}
};

template <int DT>
void launch_quantize(const MxQuantArgs& a, const MxGrid& grid, hipStream_t stream) {
  const unsigned narrow = grid.tall < 256 ? 2 * grid.tall : 0;
  if (a.codes && a.codes_t) {
    if (narrow) mx_quantize_kernel<DT, true, true, 4, 64><<<narrow, 256, 0, stream>>>(a);
    else mx_quantize_kernel<DT, true, true, 8, 128><<<grid.tall, 256, 0, stream>>>(a);
  } else if (a.codes_t) {
    if (narrow) mx_quantize_kernel<DT, false, true, 4, 64><<<narrow, 256, 0, stream>>>(a);
    else mx_quantize_kernel<DT, false, true, 8, 128><<<grid.tall, 256, 0, stream>>>(a);
  } else {
    if (grid.low) mx_quantize_kernel<DT, true, false, 2, 128><<<grid.low, 256, 0, stream>>>(a);
    else mx_quantize_kernel<DT, true, false, 8, 128><<<grid.tall, 256, 0, stream>>>(a);
  }
}

// ---------------------------------------------------------------------------
// The values back
// ---------------------------------------------------------------------------
struct MxDequantArgs {
  const uint8_t *codes, *scales;
  int64_t R, C;
  void* out;  // [R, C]
};

template <int DT, int ITER>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(MxDequantArgs a) {
  constexpr int kSize = DT == kMxF32 ? 4 : 2;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t nx = mx_slabs(a.C), ny = (a.R + 16 * ITER - 1) / (16 * ITER);
  const int64_t id = blockIdx.x, cs = id % nx, rs = id / nx % ny, z = id / nx / ny;
  const int64_t rows = mx_rows(a.R), c = cs * 128 + 8 * (lane & 15), r0 = rs * (16 * ITER) + 4 * wave + (lane >> 4);
  const uint8_t* codes = a.codes + (z * nx + cs) * rows * 64;
  const uint8_t* scales = a.scales + (z * nx + cs) * rows * 4;
  uint8_t* out = reinterpret_cast<uint8_t*>(a.out) + z * a.R * a.C * kSize;
  if (c >= a.C) return;
  uint32_t q[ITER], e[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int64_t r = r0 + 16 * i, rr = r < a.R ? r : 0;
    q[i] = *reinterpret_cast<const uint32_t*>(codes + rr * 64 + 4 * (lane & 15));
    e[i] = scales[rr * 4 + ((lane >> 2) & 3)];
  }
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int64_t r = r0 + 16 * i;
    if (r >= a.R) break;
    const float s = mx_scale_value(e[i]);
    Eight<DT> v;
    if constexpr (DT == kMxF32) {
      const floatx2 f0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], s, 0);
      const floatx2 f1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], s, 1);
      const floatx2 f2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], s, 2);
      const floatx2 f3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], s, 3);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        v.w[j] = __float_as_uint(f0[j]);
        v.w[2 + j] = __float_as_uint(f1[j]);
        v.w[4 + j] = __float_as_uint(f2[j]);
        v.w[6 + j] = __float_as_uint(f3[j]);
      }
    } else if constexpr (DT == kMxBf16) {
      const intx4 w = __builtin_bit_cast(intx4, bf16_of_codes8(q[i], s));
#pragma unroll
      for (int j = 0; j < 4; ++j) v.w[j] = (uint32_t)w[j];
    } else {
      v.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q[i], s, 0));
      v.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q[i], s, 1));
      v.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q[i], s, 2));
      v.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q[i], s, 3));
    }
    uint8_t* p = out + (r * a.C + c) * kSize;
    if (c + 8 <= a.C) {
      *reinterpret_cast<mx_intx4_any*>(p) = mx_intx4_any{(int)v.w[0], (int)v.w[1], (int)v.w[2], (int)v.w[3]};
      if constexpr (DT == kMxF32)
        *reinterpret_cast<mx_intx4_any*>(p + 16) = mx_intx4_any{(int)v.w[4], (int)v.w[5], (int)v.w[6], (int)v.w[7]};
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (c + j < a.C) {
          if constexpr (DT == kMxF32) reinterpret_cast<uint32_t*>(p)[j] = v.w[j];
          else reinterpret_cast<uint16_t*>(p)[j] = (uint16_t)(v.w[j / 2] >> (16 * (j & 1)));
        }
      }
    }
  }
}

template <int DT>
void launch_dequantize(const MxDequantArgs& a, const MxGrid& grid, hipStream_t s) {
  if (grid.low) mx_dequantize_kernel<DT, 2><<<grid.low, 256, 0, s>>>(a);
  else mx_dequantize_kernel<DT, 8><<<grid.tall, 256, 0, s>>>(a);
}

// ---------------------------------------------------------------------------
// The product, few rows
// ---------------------------------------------------------------------------
struct MxGemmArgs {
  const uint8_t *a, *as;  // [M, K] codes and scales
  const uint8_t *b, *bs;  // [N, K]
  const void* x;          // or the first operand's values, rows ldx apart, quantised on the way
  int64_t ldx;
  int64_t M, N, K;
  void* out;  // [M, N]
  int out_type;
  int share = 1 << 30;  // slabs of a work-group's share of K, where there are several
};

SFP8_DEV void store4(void* out, int type, int64_t i, const float (&v)[4], int n) {
  if (type == kMxF32) {
    float* p = reinterpret_cast<float*>(out) + i;
    if (n == 4 && ((uintptr_t)p & 15) == 0) *reinterpret_cast<floatx4*>(p) = floatx4{v[0], v[1], v[2], v[3]};
    else
      for (int j = 0; j < n; ++j) p[j] = v[j];
    return;
  }
  uint16_t* p = reinterpret_cast<uint16_t*>(out) + i;
  uint32_t w[2];
  if (type == kMxBf16) {
    w[0] = pack2_bf16(v[0], v[1]);
    w[1] = pack2_bf16(v[2], v[3]);
  } else {
    w[0] = __builtin_bit_cast(uint32_t, halfx2{(_Float16)v[0], (_Float16)v[1]});
    w[1] = __builtin_bit_cast(uint32_t, halfx2{(_Float16)v[2], (_Float16)v[3]});
  }
  if (n == 4 && ((uintptr_t)p & 7) == 0) *reinterpret_cast<intx2*>(p) = intx2{(int)w[0], (int)w[1]};
  else
    for (int j = 0; j < n; ++j) p[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
}

SFP8_DEV intx8 fp4_operand(intx4 v) { return intx8{v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }

// 16 MB rows of A times 16 NB rows of B by WV waves that share the K slabs (a
// wave takes every WV-th): the operands go from memory to registers, 16 bytes
// a lane and 1 KiB in a run, each read once in the work-group, and the waves'
// sums meet in LDS in the order of the waves.  v_mfma_scale_f32_16x16x128:
// lane l holds row l % 16, block l / 16 of a slab, and its scale; B is the
// first operand, so a lane's four sums are neighbours in a row of the output.
// XT >= 0: A is quantised here; a lane's 32 values are one block.
template <int MB, int NB, int WV, int XT>
__global__ __launch_bounds__(64 * WV) void mx_few_kernel(MxGemmArgs g) {
  __shared__ __align__(16) float red[WV][MB * 16][NB * 16 + 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, q = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NB), m0 = (int64_t)blockIdx.y * (16 * MB);
  const int64_t np = mx_rows(g.N), mp = mx_rows(g.M), S = mx_slabs(g.K);
  int64_t brow[NB], arow[MB];
#pragma unroll
  for (int j = 0; j < NB; ++j) brow[j] = (n0 + 16 * j < np ? n0 + 16 * j : np - 16) + r;
#pragma unroll
  for (int i = 0; i < MB; ++i) arow[i] = (m0 + 16 * i < mp ? m0 + 16 * i : mp - 16) + r;
  floatx4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  const auto batch = [&](auto size, int64_t s0) {  // slabs s0 and s0 + WV, or s0
    constexpr int U = decltype(size)::value, DT = XT < 0 ? 0 : XT;
    intx4 bv[U][NB], av[U][MB];
    uint32_t bsc[U][NB], asc[U][MB];
    Eight<DT> xv[U][MB][XT < 0 ? 1 : 4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t s = s0 + u * WV;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        bv[u][j] = *reinterpret_cast<const intx4*>(g.b + (s * np + brow[j]) * 64 + 16 * q);
        bsc[u][j] = *reinterpret_cast<const uint32_t*>(g.bs + (s * np + brow[j]) * 4);
      }
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        if constexpr (XT < 0) {
          av[u][i] = *reinterpret_cast<const intx4*>(g.a + (s * mp + arow[i]) * 64 + 16 * q);
          asc[u][i] = *reinterpret_cast<const uint32_t*>(g.as + (s * mp + arow[i]) * 4);
        } else {
          const int64_t k = s * 128 + 32 * q, left = arow[i] < g.M ? g.K - k : 0, at = arow[i] * g.ldx + k;
          if (left >= 32) {
#pragma unroll
            for (int c = 0; c < 4; ++c) xv[u][i][c] = load8<DT>(g.x, at + 8 * c);
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              xv[u][i][c] = Eight<DT>{};
              if (left > 8 * c) xv[u][i][c] = load8_upto<DT>(g.x, at + 8 * c, left - 8 * c);
            }
          }
        }
      }
    }
    if constexpr (U > 1) __builtin_amdgcn_sched_barrier(0);  // the loads stay ahead of the products
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        if constexpr (XT >= 0) {
          uint32_t m = abs_max8<DT>(xv[u][i][0]);
#pragma unroll
          for (int c = 1; c < 4; ++c) m = max_u(m, abs_max8<DT>(xv[u][i][c]));
          asc[u][i] = mx_scale_code(abs_bits_to_f32<DT>(m)) << (8 * q);
          const float sv = mx_scale_value(asc[u][i] >> (8 * q));
#pragma unroll
          for (int c = 0; c < 4; ++c) av[u][i][c] = (int)codes8<DT>(xv[u][i][c], sv);
        }
      }
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
              fp4_operand(bv[u][j]), fp4_operand(av[u][i]), acc[i][j], 4, 4, 0, (int)(bsc[u][j] >> (8 * q)), 0,
              (int)(asc[u][i] >> (8 * q)));
    }
  };
  // Two slabs at once pay with many operands a slab, whose loads the compiler otherwise spreads over the products
  // (1024 x 1024 x 4096 9.4 -> 8.1 us); the small variants lose by it (8 x 8192 x 2048 from bf16 rows 5.4 against 5.7).
  const int64_t n = (S - wave + WV - 1) / WV;  // this wave's slabs
  int64_t i = 0;
  if constexpr (MB * NB >= 8) {
    for (; i + 2 <= n; i += 2) batch(std::integral_constant<int, 2>{}, wave + i * WV);
    for (; i < n; ++i) batch(std::integral_constant<int, 1>{}, wave + i * WV);
  } else {
#pragma unroll 2
    for (; i < n; ++i) batch(std::integral_constant<int, 1>{}, wave + i * WV);
  }
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) *reinterpret_cast<floatx4*>(&red[wave][16 * i + r][16 * j + 4 * q]) = acc[i][j];
  __syncthreads();
  for (int u = tid; u < MB * 16 * NB * 4; u += 64 * WV) {
    const int m = u / (NB * 4), n = 4 * (u % (NB * 4));
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WV; ++w) {
      const floatx4 p = *reinterpret_cast<const floatx4*>(&red[w][m][n]);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += p[j];
    }
    const int64_t left = g.N - (n0 + n);
    if (m0 + m < g.M && left > 0) store4(g.out, g.out_type, (m0 + m) * g.N + n0 + n, v, left < 4 ? (int)left : 4);
  }
}

// ---------------------------------------------------------------------------
// The product, tiles
// ---------------------------------------------------------------------------
// TM x TM outputs of one work-group: 8 waves of 128 x 64 (TM = 256) or 4 of 64 x
// 64 (TM = 128, two work-groups a CU).  K advances a slab (128 values, 64 bytes
// of a row) at a time through a ring of four LDS stages: codes of TM rows of A
// and of B, and their four scales a row.  Everything comes by DMA
// (buffer_load .. lds, 1 KiB of codes or 256 bytes of scales a wave and
// instruction), three stages ahead; rows past the operand's end read as zeros.
// Row r keeps its 16-byte chunk c at c ^ (r / 4) % 4: the 16 rows that a lane
// group reads lie in different banks.
//
// v_mfma_scale_f32_32x32x64: lane l holds row l % 32 and 32 values, which are
// one block of the row: half g = l / 32 takes chunk 2 g + h in step h of the two
// of a slab, and its scale is byte 2 g + h of the row's four.  B is the first
// operand, and its rows are permuted as they are fetched so that a lane's 16
// sums of a block are neighbours: columns 32 g + 16 nb + v of the wave's 64.
//
// A stage's MFMAs run in a fixed order with the next stage's LDS reads and the
// DMA between them; the first two go ahead of the stage's wait and barrier.
template <int TM>
struct MxTile {
  static constexpr int TB = TM == 256 ? 4 : 2, NB = 2, WN = TM / 64, kWaves = 2 * WN, kStages = 4;
  static constexpr int kSide = TM * 64, kScaleSide = TM * 4;        // bytes of a stage, one operand
  static constexpr int kStage = 2 * kSide + 2 * kScaleSide, kLds = kStages * kStage;
  static constexpr int kCodeDma = TM / 16 / kWaves;                  // of A, and of B, a wave and stage: 2
  static constexpr int kDma = 2 * kCodeDma + 1;                      // and one of scales: 64 rows a wave
  static constexpr int kMfma = 2 * TB * NB;
  static_assert(kCodeDma == 2 && kWaves * 64 == 2 * TM, "one scale instruction a wave");
  using Rsrc = __amdgpu_buffer_rsrc_t;
  using Lds = __attribute__((address_space(3))) void*;

  struct Frag {
    intx4 a[TB][2], b[NB][2];
    uint32_t as[TB], bs[NB];
  };
  typedef floatx16 Acc[TB][NB];

  struct Operands {
    const uint8_t *a, *b, *scales;       // this tile's first rows of the first slab; scales of A or of B by wave
    int64_t a_step, b_step, scale_step;  // bytes from slab to slab
    int a_bytes, b_bytes, scale_bytes;   // of the tile's rows that there are
    int stages;
  };
  uint8_t* lds;
  Operands op;
  uint32_t va[2], vb[2], vs;      // DMA lane offsets
  uint32_t da[2], db[2], ds;      // and where in a stage they land
  uint32_t ra[2], rb[2], rs, rt;  // LDS read offsets: chunk 2 g + h of A and B, scales of A and B

  static SFP8_DEV Rsrc rsrc(const uint8_t* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), (short)0, bytes, 0x00020000);
  }
  // column of the wave's 64 that row i of block nb stands for
  static SFP8_DEV int column(int p) {
    const int nb = (p >> 5) & 1, i = p & 31;
    return (p & ~63) + 32 * ((i >> 2) & 1) + 16 * nb + 4 * (i >> 3) + (i & 3);
  }

  SFP8_DEV MxTile(uint8_t* l, const Operands& o) : lds(l), op(o) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % 2, wn = wave / 2;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = 32 * wave + 16 * j + (lane >> 2);
      const uint32_t chunk = (uint32_t)(((lane & 3) ^ ((r >> 2) & 3)) << 4);
      va[j] = (uint32_t)r * 64 + chunk;
      vb[j] = (uint32_t)column(r) * 64 + chunk;
      da[j] = (uint32_t)(32 * wave + 16 * j) * 64;
      db[j] = kSide + da[j];
    }
    const bool of_b = wave >= WN;
    const int r = 64 * (of_b ? wave - WN : wave) + lane;
    vs = (uint32_t)(of_b ? column(r) : r) * 4;
    ds = 2 * kSide + (uint32_t)wave * 256;
    const int fr = lane & 31, g = lane >> 5, sw = (fr >> 2) & 3;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t chunk = (uint32_t)(((2 * g + h) ^ sw) << 4);
      ra[h] = (uint32_t)(32 * TB * wm + fr) * 64 + chunk;
      rb[h] = kSide + (uint32_t)(64 * wn + fr) * 64 + chunk;
    }
    rs = 2 * kSide + (uint32_t)(32 * TB * wm + fr) * 4 + 2 * g;
    rt = 2 * kSide + kScaleSide + (uint32_t)(64 * wn + fr) * 4 + 2 * g;
  }

  // DMA instruction j of stage s into ring slot `slot`; past the last stage nothing is read
  SFP8_DEV void dma(int j, int s, int slot) const {
    const bool live = s < op.stages;
    uint8_t* at = lds + slot * kStage;
    if (j < 2)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc(op.a + s * op.a_step, live ? op.a_bytes : 0), (Lds)(at + da[j]), 16,
                                               va[j], 0, 0, 0);
    else if (j < 4)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc(op.b + s * op.b_step, live ? op.b_bytes : 0),
                                               (Lds)(at + db[j - 2]), 16, vb[j - 2], 0, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc(op.scales + s * op.scale_step, live ? op.scale_bytes : 0),
                                               (Lds)(at + ds), 4, vs, 0, 0, 0);
  }
  // Fragment i: A block i, or B block i - TB, with its scales
  template <int I>
  SFP8_DEV void read(int slot, Frag& f) const {
    const uint8_t* at = lds + slot * kStage;
    if constexpr (I < TB) {
#pragma unroll
      for (int h = 0; h < 2; ++h) f.a[I][h] = *reinterpret_cast<const intx4*>(at + ra[h] + I * 32 * 64);
      f.as[I] = *reinterpret_cast<const uint16_t*>(at + rs + I * 32 * 4);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) f.b[I - TB][h] = *reinterpret_cast<const intx4*>(at + rb[h] + (I - TB) * 32 * 64);
      f.bs[I - TB] = *reinterpret_cast<const uint16_t*>(at + rt + (I - TB) * 32 * 4);
    }
  }
  template <int I = 0>
  SFP8_DEV void read_all(int slot, Frag& f) const {
    if constexpr (I < TB + NB) {
      read<I>(slot, f);
      read_all<I + 1>(slot, f);
    }
  }
  template <int I>
  static SFP8_DEV void mfma(const Frag& f, Acc& acc) {
    constexpr int h = I / (TB * NB), tb = I / NB % TB, nb = I % NB;
    acc[tb][nb] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fp4_operand(f.b[nb][h]), fp4_operand(f.a[tb][h]),
                                                                  acc[tb][nb], 4, 4, h, (int)f.bs[nb], h,
                                                                  (int)f.as[tb]);
  }
  template <int LO, int HI>
  static SFP8_DEV void mfmas(const Frag& f, Acc& acc) {
    if constexpr (LO < HI) {
      mfma<LO>(f, acc);
      mfmas<LO + 1, HI>(f, acc);
    }
  }
  // MFMA I, then a fragment of the next stage and DMA instruction D (either may be -1)
  template <int I, int R, int D>
  SFP8_DEV void slot(const Frag& cur, Frag& nxt, Acc& acc, int s, int read_slot, int dma_slot) const {
    mfma<I>(cur, acc);
    if constexpr (R >= 0) read<R>(read_slot, nxt);
    if constexpr (D >= 0) dma(D, s + kStages - 1, dma_slot);
    __builtin_amdgcn_sched_barrier(0);
  }
  // Stage s on `cur`: reads stage s + 1 into `nxt`, fetches stage s + 3 into the slot of stage s - 1.
  SFP8_DEV void stage(const Frag& cur, Frag& nxt, Acc& acc, int s) const {
    const int rd = (s + 1) % kStages, wr = (s + kStages - 1) % kStages;
    mfmas<0, 2>(cur, acc);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(kDma * (kStages - 3)) : "memory");
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (TB == 4) {
      slot<2, 0, -1>(cur, nxt, acc, s, rd, wr);
      slot<3, -1, 0>(cur, nxt, acc, s, rd, wr);
      slot<4, 4, -1>(cur, nxt, acc, s, rd, wr);
      slot<5, -1, 1>(cur, nxt, acc, s, rd, wr);
      slot<6, 5, -1>(cur, nxt, acc, s, rd, wr);
      slot<7, -1, 2>(cur, nxt, acc, s, rd, wr);
      slot<8, 1, -1>(cur, nxt, acc, s, rd, wr);
      slot<9, -1, 3>(cur, nxt, acc, s, rd, wr);
      slot<10, 2, -1>(cur, nxt, acc, s, rd, wr);
      slot<11, -1, 4>(cur, nxt, acc, s, rd, wr);
      slot<12, 3, -1>(cur, nxt, acc, s, rd, wr);
      mfmas<13, 16>(cur, acc);
    } else {
      slot<2, 0, 0>(cur, nxt, acc, s, rd, wr);
      slot<3, 2, 1>(cur, nxt, acc, s, rd, wr);
      slot<4, 3, 2>(cur, nxt, acc, s, rd, wr);
      slot<5, 1, 3>(cur, nxt, acc, s, rd, wr);
      slot<6, -1, 4>(cur, nxt, acc, s, rd, wr);
      mfmas<7, 8>(cur, acc);
    }
    __builtin_amdgcn_sched_barrier(0);
  }

  SFP8_DEV void run(Acc& acc) const {
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j)
        acc[i][j] = floatx16{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s)
#pragma unroll
      for (int j = 0; j < kDma; ++j) dma(j, s, s);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(kDma * (kStages - 2)) : "memory");
    Frag f0, f1;
    read_all(0, f0);
    // two stages a turn, so that the fragments alternate by name; an odd count runs one more on zeros
    for (int s = 0; s < op.stages; s += 2) {
      stage(f0, f1, acc, s);
      stage(f1, f0, acc, s + 1);
    }
    // nothing in flight into the ring, and nobody reads it any more
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
  }
};

// Tiles in the order in which work-groups take them: the 8 XCDs own runs of
// them, each 8 tile rows high, so that an XCD's L2 serves the columns again.
SFP8_DEV bool mx_tile_of(int id, int rows, int cols, int& r, int& c) {
  const int n = rows * cols, per = (n + 7) / 8;
  const int t = (id & 7) * per + (id >> 3);
  if ((id >> 3) >= per || t >= n) return false;
  const int first = t / (8 * cols) * 8, high = rows - first < 8 ? rows - first : 8, in = t - first * cols;
  r = first + in % high;
  c = in / high;
  return true;
}

// 8 neighbours of an output row from element i on, `left` of them in the matrix.
template <int OUT>
SFP8_DEV void store8(void* out, int64_t i, const Eight<OUT>& v, int64_t left) {
  if constexpr (OUT == kMxF32) {
    typedef int any4 __attribute__((ext_vector_type(4), aligned(4)));
    float* p = reinterpret_cast<float*>(out) + i;
    if (left >= 8) {
      *reinterpret_cast<any4*>(p) = any4{(int)v.w[0], (int)v.w[1], (int)v.w[2], (int)v.w[3]};
      *reinterpret_cast<any4*>(p + 4) = any4{(int)v.w[4], (int)v.w[5], (int)v.w[6], (int)v.w[7]};
    } else {
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < left) p[j] = __uint_as_float(v.w[j]);
    }
  } else {
    uint16_t* p = reinterpret_cast<uint16_t*>(out) + i;
    if (left >= 8) {
      *reinterpret_cast<mx_intx4_any*>(p) = mx_intx4_any{(int)v.w[0], (int)v.w[1], (int)v.w[2], (int)v.w[3]};
    } else {
#pragma unroll
      for (int j = 0; j < 7; ++j)
        if (j < left) p[j] = (uint16_t)(v.w[j / 2] >> (16 * (j & 1)));
    }
  }
}

// A wave's 32 TB x 64 sums to memory: through its own part of the LDS (the ring
// is done with), so that each store writes whole 128-byte lines: eight lanes a
// row.  16-byte chunk c of row r lies at c ^ (r / 2) % 8.  ROWS of them at a time.
template <int OUT, int TB, int ROWS>
SFP8_DEV void store_wave(uint8_t* lds, void* out, int64_t m, int64_t n, int64_t M, int64_t N,
                         const floatx16 (&acc)[TB][2]) {
  constexpr int kSize = OUT == kMxF32 ? 4 : 2, kRow = 64 * kSize, kChunks = kRow / 16;
  const int lane = threadIdx.x & 63, g = lane >> 5;
#pragma unroll
  for (int b0 = 0; b0 < TB; b0 += ROWS / 32) {
#pragma unroll
    for (int b = 0; b < ROWS / 32; ++b) {
      const int r = 32 * b + (lane & 31);
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
        const floatx16& v = acc[b0 + b][nb];
#pragma unroll
        for (int c = 0; c < kSize; ++c) {  // 16 values are kSize chunks
          intx4 w;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (OUT == kMxF32) w[j] = (int)__float_as_uint(v[4 * c + j]);
            else if constexpr (OUT == kMxBf16) w[j] = (int)pack2_bf16(v[8 * c + 2 * j], v[8 * c + 2 * j + 1]);
            else
              w[j] = __builtin_bit_cast(int, halfx2{(_Float16)v[8 * c + 2 * j], (_Float16)v[8 * c + 2 * j + 1]});
          }
          const int chunk = (32 * g + 16 * nb) * kSize / 16 + c;
          *reinterpret_cast<intx4*>(lds + r * kRow + 16 * ((chunk & ~7) | ((chunk ^ (r >> 1)) & 7))) = w;
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int i = 0; i < ROWS / 8; ++i) {
      const int r = 8 * i + (lane >> 3), c = lane & 7;  // eight values a lane
      Eight<OUT> v;
#pragma unroll
      for (int j = 0; j < kChunks / 8; ++j) {
        const int chunk = c * (kChunks / 8) + j;
        const intx4 w =
            *reinterpret_cast<const intx4*>(lds + r * kRow + 16 * ((chunk & ~7) | ((chunk ^ (r >> 1)) & 7)));
#pragma unroll
        for (int k = 0; k < 4; ++k) v.w[4 * j + k] = (uint32_t)w[k];
      }
      const int64_t row = m + 32 * b0 + r;
      if (row < M) store8<OUT>(out, row * N + n + 8 * c, v, N - n - 8 * c);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// Sums of a share of K, [M, N] fp32, so many values after those of the share before
inline __host__ __device__ int64_t mx_part(int64_t M, int64_t N) { return (M * N + 3) / 4 * 4; }

// gridDim.y work-groups share the slabs of a tile; with more than one the results are their sums alone (fp32).
template <int TM, int OUT>
__global__ __launch_bounds__(2 * TM, 2) void mx_tile_kernel(MxGemmArgs g) {
  using Tile = MxTile<TM>;
  __shared__ __align__(1024) uint8_t lds[Tile::kLds];
  const int64_t mp = mx_rows(g.M), np = mx_rows(g.N);
  int tr, tc;
  if (!mx_tile_of(blockIdx.x, (int)((mp + TM - 1) / TM), (int)((np + TM - 1) / TM), tr, tc)) return;
  const int64_t m0 = (int64_t)tr * TM, n0 = (int64_t)tc * TM;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int arows = (int)(mp - m0 < TM ? mp - m0 : TM), brows = (int)(np - n0 < TM ? np - n0 : TM);
  const bool of_b = wave >= Tile::WN;
  const int64_t sp = of_b ? np : mp;
  const int slabs = (int)mx_slabs(g.K), lo = min((int)blockIdx.y * g.share, slabs), hi = min(lo + g.share, slabs);
  const typename Tile::Operands op{
      g.a + (lo * mp + m0) * 64, g.b + (lo * np + n0) * 64,
      of_b ? g.bs + (lo * np + n0) * 4 : g.as + (lo * mp + m0) * 4, mp * 64, np * 64, sp * 4,
      arows * 64, brows * 64, (of_b ? brows : arows) * 4, hi - lo};
  typename Tile::Acc acc;
  Tile(lds, op).run(acc);
  constexpr int kPart = Tile::kLds / Tile::kWaves & ~1023, kRow = 64 * (OUT == kMxF32 ? 4 : 2);
  constexpr int kRows = kPart / kRow / 32 * 32 < 32 * Tile::TB ? (kPart / kRow >= 64 ? 64 : 32) : 32 * Tile::TB;
  void* out = g.out;
  if constexpr (OUT == kMxF32) out = reinterpret_cast<float*>(g.out) + blockIdx.y * mx_part(g.M, g.N);
  store_wave<OUT, Tile::TB, kRows>(lds + wave * kPart, out, m0 + 32 * Tile::TB * (wave % 2), n0 + 64 * (wave / 2),
                                   g.M, g.N, acc);
}

// The shares' sums in order, and the one rounding.
__global__ __launch_bounds__(256) void mx_sum_kernel(const float* parts, int shares, int64_t n, void* out, int type) {
  const int64_t i = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x), step = (n + 3) / 4 * 4;
  if (i >= n) return;
  floatx4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int y = 0; y < shares; ++y) {
    const floatx4 p = *reinterpret_cast<const floatx4*>(parts + y * step + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += p[j];
  }
  store4(out, type, i, {v[0], v[1], v[2], v[3]}, n - i < 4 ? (int)(n - i) : 4);
}

void launch_shares(const MxGemmArgs& g, int64_t tiles, int shares, void* ws, hipStream_t s) {
  MxGemmArgs p = g;
  p.out = ws;
  p.share = (int)((mx_slabs(g.K) + shares - 1) / shares);
  mx_tile_kernel<128, kMxF32><<<dim3((unsigned)((tiles + 7) / 8 * 8), (unsigned)shares), 256, 0, s>>>(p);
  mx_sum_kernel<<<(unsigned)((g.M * g.N + 1023) / 1024), 256, 0, s>>>((const float*)ws, shares, g.M * g.N, g.out,
                                                                      g.out_type);
}

template <int TM>
void launch_tiles(const MxGemmArgs& g, int64_t tiles, hipStream_t s) {
  const unsigned grid = (unsigned)((tiles + 7) / 8 * 8);
  if (g.out_type == kMxF32) mx_tile_kernel<TM, kMxF32><<<grid, 2 * TM, 0, s>>>(g);
  else if (g.out_type == kMxBf16) mx_tile_kernel<TM, kMxBf16><<<grid, 2 * TM, 0, s>>>(g);
  else mx_tile_kernel<TM, kMxF16><<<grid, 2 * TM, 0, s>>>(g);
}

template <int MB, int NB, int WV, int XT>
void launch_few(const MxGemmArgs& g, hipStream_t s) {
  const dim3 grid((unsigned)((g.N + 16 * NB - 1) / (16 * NB)), (unsigned)((g.M + 16 * MB - 1) / (16 * MB)));
  mx_few_kernel<MB, NB, WV, XT><<<grid, 64 * WV, 0, s>>>(g);
}

inline int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}
inline bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
inline bool type_ok(int dtype) { return dtype >= kMxF32 && dtype <= kMxF16; }
constexpr int64_t kMxMaxDim = (int64_t)1 << 31;

// By the number of tiles (us; M, N, K):
//  256 x 256 where they fill the CUs and K is long: its loop fetches half of what that of 128 x 128 does for a
//  product, which hides its stores behind a second work-group: 16384, 8192, 4096 281 against 362; 4096, 4096, 2560
//  26.3 against 28.3; but 16384, 4096, 2048 96.5 against 88.8 and 65536, 1024, 1024 72.0 against 55.5.
//  128 x 128 from half a tile a CU on (1003, 2050, 1000 6.1 against 10.6; 512, 4096, 4096 11.1 against 13.2);
//  below that the waves share K (1024, 1024, 4096 8.1 against 10.6).
//  Where K is very long (the weight gradients of many tokens) work-groups share it, 128 x 128 each, until there is
//  one a CU with at least 4096 of K: 1024, 1024, 65536 74 -> 54; 1000, 1030, 16384 40 -> 25; 512, 1536, 49152 77 -> 34;
//  the sums' way through memory costs more than it gives at 1024, 1024, 12288 (18.0, shared 20.6; 16384 23.0, 24.0),
//  512, 512, 24576 (15.8, 17.2) and 256, 256, 32768 (13.6, 15.4), but not at 128, 128, 65536 (24.2, 16.9).
//  Tiles count whole, also where M or N fills a part of them alone, and the limits come of the sizes above, wide in
//  both.  A few rows by very many columns, in a graph (us): 128 x 128 wins from N = 65536 on, also for one row (1,
//  65536, 2048 15.7, 16 x 32 17.2; 64, 131072, 2048 36.4, 64 x 64 40.9), and loses at 16384 (8, 16384, 2048 8.2, 16 x
//  32 5.8; 64, 16384, 4096 12.8, 64 x 64 10.4; 16384, 16, 8192 20.4, 64 x 32 13.9); 256 x 256, which the rule takes
//  there for a long K, loses to 128 x 128 (8, 131072, 4096 59.4 and 53.5; 64, 65536, 4096 38.0 and 36.4).
struct MxPlan {
  int tile = 0, shares = 1;  // 0: by waves that share K
  MxPlan(int64_t M, int64_t N, int64_t K) {
    const auto tiles = [&](int64_t n) { return ((M + n - 1) / n) * ((N + n - 1) / n); };
    if (tiles(256) >= 256 && K >= 2560) {
      tile = 256;
    } else if (tiles(128) <= 128 && K >= 16384 && (K >= 49152 || M * N >= ((int64_t)1 << 33) / K)) {
      const int64_t fill = 256 / tiles(128), most = K / 4096;
      tile = 128, shares = (int)(fill < most ? fill : most);
    } else if (tiles(128) >= 128) {
      tile = 128;
    }
  }
  int64_t workspace(int64_t M, int64_t N) const { return shares > 1 ? shares * mx_part(M, N) * 4 : 0; }
};

constexpr int64_t kMxMaxTiles = ((int64_t)1 << 24) - 8;  // of 256 threads: a grid has less than 2^32
constexpr int64_t kMxMaxTiles256 = ((int64_t)1 << 23) - 8;  // of 512
constexpr int64_t kMxMaxRowsN = ((int64_t)1 << 27) - 16;  // 16 columns of 512 threads

}  // namespace sfp8

using namespace sfp8;

extern "C" {

int64_t sfp8_mxfp4_code_bytes(int64_t R, int64_t C) {
  return R < 0 || C < 0 || R > kMxMaxDim || C > kMxMaxDim ? -1 : mx_slabs(C) * mx_rows(R) * 64;
}

int sfp8_mxfp4_quantize(const void* x, int dtype, int64_t batch, int64_t R, int64_t C, int64_t ld,
                        int64_t batch_stride, void* codes, void* scales, void* codes_t, void* scales_t, void* stream) {
  if (!type_ok(dtype) || batch < 0 || R < 0 || C < 0 || R > kMxMaxDim || C > kMxMaxDim || ld < 0 || batch_stride < 0)
    return kErrBadShape;
  if (!codes != !scales || !codes_t != !scales_t) return kErrNullPointer;
  if (batch == 0 || R == 0 || C == 0 || (!codes && !codes_t)) return kOk;
  if (!x) return kErrNullPointer;
  if (!aligned(x, dtype == kMxF32 ? 4 : 2) || !aligned(codes, 16) || !aligned(codes_t, 16) || !aligned(scales, 4) ||
      !aligned(scales_t, 4))
    return kErrBadAlignment;
  const int64_t tiles = mx_slabs(C) * ((R + 127) / 128);
  if (tiles > kMxMaxTiles / batch) return kErrBadShape;
  const MxQuantArgs a{x, R, C, ld, batch_stride, (uint8_t*)codes, (uint8_t*)scales, (uint8_t*)codes_t,
                      (uint8_t*)scales_t};
  const MxGrid grid(batch, R, C);
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == kMxF32) launch_quantize<kMxF32>(a, grid, s);
  else if (dtype == kMxBf16) launch_quantize<kMxBf16>(a, grid, s);
  else launch_quantize<kMxF16>(a, grid, s);
  return launched();
}

int sfp8_mxfp4_dequantize(const void* codes, const void* scales, int64_t batch, int64_t R, int64_t C, void* out,
                          int dtype, void* stream) {
  if (!type_ok(dtype) || batch < 0 || R < 0 || C < 0 || R > kMxMaxDim || C > kMxMaxDim) return kErrBadShape;
  if (batch == 0 || R == 0 || C == 0) return kOk;
  if (!codes || !scales || !out) return kErrNullPointer;
  if (!aligned(codes, 16) || !aligned(scales, 4) || !aligned(out, 16)) return kErrBadAlignment;
  const int64_t tiles = mx_slabs(C) * ((R + 127) / 128);
  if (tiles > kMxMaxTiles / batch) return kErrBadShape;
  const MxDequantArgs a{(const uint8_t*)codes, (const uint8_t*)scales, R, C, out};
  const MxGrid grid(batch, R, C);
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == kMxF32) launch_dequantize<kMxF32>(a, grid, s);
  else if (dtype == kMxBf16) launch_dequantize<kMxBf16>(a, grid, s);
  else launch_dequantize<kMxF16>(a, grid, s);
  return launched();
}

int64_t sfp8_mxfp4_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 0 || N < 0 || K < 0 || M > kMxMaxDim || N > kMxMaxDim || K > kMxMaxDim) return -1;
  return M == 0 || N == 0 ? 0 : MxPlan(M, N, K).workspace(M, N);
}

int sfp8_mxfp4_gemm(const void* a, const void* a_scales, const void* b, const void* b_scales, int64_t M, int64_t N,
                    int64_t K, void* out, int dtype, void* ws, int64_t ws_bytes, void* stream) {
  if (!type_ok(dtype) || M < 0 || N < 0 || K < 0 || M > kMxMaxDim || N > kMxMaxDim || K > kMxMaxDim)
    return kErrBadShape;
  if (M == 0 || N == 0) return kOk;
  if (!out || (K && (!a || !a_scales || !b || !b_scales))) return kErrNullPointer;
  if (!aligned(a, 16) || !aligned(b, 16) || !aligned(a_scales, 4) || !aligned(b_scales, 4) || !aligned(out, 16))
    return kErrBadAlignment;
  const MxGemmArgs g{(const uint8_t*)a, (const uint8_t*)a_scales, (const uint8_t*)b, (const uint8_t*)b_scales,
                     nullptr, 0, M, N, K, out, dtype};
  const hipStream_t st = (hipStream_t)stream;
  // Without tiles, in the largest block of which there are 256 (us): 64, 4096, 4096 32 x 32 4.7, 16 x 16 6.7, 64 x 64
  // 8.5; 128, 1024, 8192 16 x 32 5.4, 64 x 64 12.4.
  const auto tiles = [&](int64_t m, int64_t n) { return ((M + m - 1) / m) * ((N + n - 1) / n); };
  if (tiles(128, 128) > kMxMaxTiles) return kErrBadShape;
  const MxPlan plan(M, N, K);
  if (plan.tile == 256 && tiles(256, 256) > kMxMaxTiles256) return kErrBadShape;
  if (plan.shares > 1) {
    if (!ws) return kErrNullPointer;
    if (!aligned(ws, 16)) return kErrBadAlignment;
    if (ws_bytes < plan.workspace(M, N)) return kErrWorkspaceTooSmall;
  }
  if (plan.tile == 256) launch_tiles<256>(g, tiles(256, 256), st);
  else if (plan.shares > 1) launch_shares(g, tiles(128, 128), plan.shares, ws, st);
  else if (plan.tile == 128) launch_tiles<128>(g, tiles(128, 128), st);
  else if (tiles(64, 64) >= 256) launch_few<4, 4, 4, -1>(g, st);
  else if (M > 32 && tiles(64, 32) >= 256) launch_few<4, 2, 8, -1>(g, st);
  else if (M > 16 && tiles(32, 32) >= 256) launch_few<2, 2, 8, -1>(g, st);
  else if (tiles(16, 32) >= 256) launch_few<1, 2, 8, -1>(g, st);
  else launch_few<1, 1, 8, -1>(g, st);
  return launched();
}

int sfp8_mxfp4_gemm_rows(const void* x, int x_type, int64_t ldx, const void* b, const void* b_scales, int64_t M,
                         int64_t N, int64_t K, void* out, int dtype, void* stream) {
  if (!type_ok(dtype) || !type_ok(x_type) || M < 0 || M > 16 || N < 0 || K < 0 || N > kMxMaxRowsN ||
      K > kMxMaxDim || ldx < 0)
    return kErrBadShape;
  if (M == 0 || N == 0) return kOk;
  if (!out || (K && (!x || !b || !b_scales))) return kErrNullPointer;
  if (!aligned(x, x_type == kMxF32 ? 4 : 2) || !aligned(b, 16) || !aligned(b_scales, 4) || !aligned(out, 16))
    return kErrBadAlignment;
  const MxGemmArgs g{nullptr, nullptr, (const uint8_t*)b, (const uint8_t*)b_scales, x, ldx, M, N, K, out, dtype};
  const hipStream_t s = (hipStream_t)stream;
  if (x_type == kMxF32) launch_few<1, 1, 8, kMxF32>(g, s);
  else if (x_type == kMxBf16) launch_few<1, 1, 8, kMxBf16>(g, s);
  else launch_few<1, 1, 8, kMxF16>(g, s);
  return launched();
}

}  // extern "C"
