// Routing of tokens to experts (gfx950): what runs around the grouped expert
// kernels of a mixture-of-experts layer.
//
//  * moe_route: from the router's logits to each token's top_k experts and
//    their weights (softmax or sigmoid scores, a bias that only the order
//    sees, groups of experts, renormalised weights), and its backward pass
//  * moe_expert_order: the stable order of the (token, slot) pairs by expert
//    that the grouped kernels read (moe.hip: "expert-order rows")
//  * moe_combine: the weighted sum of each token's expert rows, and the
//    gradients of the rows and of the weights
//
// None of these has matrix work: each is bound by the bytes it reads and
// writes, or, for few tokens, by its launches.
#include "common.h"

namespace sfp8 {

constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxK = 64;
enum : int { kF32 = 0, kBf16 = 1, kF16 = 2 };
enum : int { kSoftmax = 0, kSigmoid = 1 };

SFP8_DEV float half_bits_to_f32(uint32_t b) { return (float)__builtin_bit_cast(_Float16, (uint16_t)b); }
SFP8_DEV uint32_t f32_to_half_bits(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }

SFP8_DEV float load_as_f32(const void* p, int dtype, int64_t i) {
  if (dtype == kF32) return reinterpret_cast<const float*>(p)[i];
  const uint32_t b = reinterpret_cast<const uint16_t*>(p)[i];
  return dtype == kBf16 ? bf16_bits_to_f32(b) : half_bits_to_f32(b);
}
SFP8_DEV void store_f32_as(void* p, int dtype, int64_t i, float v) {
  if (dtype == kF32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(dtype == kBf16 ? f32_to_bf16_bits(v) : f32_to_half_bits(v));
}

// The order of two order values: NaN above everything, then by value.
SFP8_DEV bool ranks_above(double a, double b) { return a > b || (a != a && b == b); }

SFP8_DEV double wave_max_nan_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const double w = __shfl_xor(v, o, 64);
    v = ranks_above(w, v) ? w : v;
  }
  return v;
}

struct RouteArgs {
  const void* logits;
  int dtype;
  int64_t T, ld;
  int E, k, score, groups, top_groups, group_best, renorm;
  float scale;
  const float* bias;
  const uint8_t* mask;
  float* weights;
  int64_t* selected;
  float* picked;
};

// One wave per token, everything in 64 bits: v[e] is the order value of
// expert e (LDS), -inf where it cannot be taken (any more).
__global__ __launch_bounds__(256) void moe_route_kernel(const RouteArgs a) {
  extern __shared__ __align__(16) double lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * 4 + wave;
  if (t >= a.T) return;
  double* v = lds + (int64_t)wave * a.E;
  const double ninf = -__builtin_inf();
  const int64_t row = t * a.ld;
  if (a.mask && !a.mask[t]) {
    if (lane < a.k) {
      a.weights[t * a.k + lane] = 0.0f;
      a.selected[t * a.k + lane] = -1;
      if (a.picked) a.picked[t * a.k + lane] = 0.0f;
    }
    return;
  }
  double m = 0.0, z = 1.0;
  if (a.score == kSoftmax) {
    m = ninf;
    for (int e = lane; e < a.E; e += 64) {
      const double l = load_as_f32(a.logits, a.dtype, row + e);
      m = ranks_above(l, m) ? l : m;
    }
    m = wave_max_nan_f64(m);
    z = 0.0;
    for (int e = lane; e < a.E; e += 64) z += exp((double)load_as_f32(a.logits, a.dtype, row + e) - m);
    z = wave_sum_f64(z);
  }
  const auto score_of = [&](double l) { return a.score == kSoftmax ? exp(l - m) / z : 1.0 / (1.0 + exp(-l)); };
  for (int e = lane; e < a.E; e += 64) {
    const double l = load_as_f32(a.logits, a.dtype, row + e);
    v[e] = l == ninf ? ninf : a.bias ? score_of(l) + (double)a.bias[e] : l;
  }
  __builtin_amdgcn_wave_barrier();
  if (a.groups > 1) {
    const int gs = a.E / a.groups;
    double g = ninf;  // the value of group `lane`
    if (lane < a.groups) {
      double b1 = ninf, b2 = ninf;
      for (int e = lane * gs; e < lane * gs + gs; ++e) {
        const double x = v[e];
        if (ranks_above(x, b1)) {
          b2 = b1;
          b1 = x;
        } else if (ranks_above(x, b2)) {
          b2 = x;
        }
      }
      if (a.group_best == 1 || b1 == ninf) {
        g = b1;
      } else if (a.bias) {
        g = b1 + (b2 == ninf ? 0.0 : b2);
      } else {
        g = score_of(b1) + (b2 == ninf ? 0.0 : score_of(b2));
      }
    }
    int rank = 0;
    for (int j = 0; j < a.groups; ++j) {
      const double o = __shfl(g, j, 64);
      rank += ranks_above(o, g) || (j < lane && !ranks_above(g, o));
    }
    if (lane < a.groups && (g == ninf || rank >= a.top_groups))
      for (int e = lane * gs; e < lane * gs + gs; ++e) v[e] = ninf;
    __builtin_amdgcn_wave_barrier();
  }
  int mine = -1;  // the expert of slot `lane`
  for (int s = 0; s < a.k; ++s) {
    double best = ninf;
    int at = a.E;
    for (int e = lane; e < a.E; e += 64) {
      const double x = v[e];
      if (ranks_above(x, best)) {
        best = x;
        at = e;
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const double ob = __shfl_xor(best, o, 64);
      const int oa = __shfl_xor(at, o, 64);
      if (ranks_above(ob, best) || (!ranks_above(best, ob) && oa < at)) {
        best = ob;
        at = oa;
      }
    }
    if (best == ninf) break;
    if (lane == s) mine = at;
    if (lane == 0) v[at] = ninf;
    __builtin_amdgcn_wave_barrier();
  }
  const bool live = lane < a.k && mine >= 0;
  const double l = live ? (double)load_as_f32(a.logits, a.dtype, row + mine) : ninf;
  double w = 0.0;
  if (!a.renorm) {
    w = live ? score_of(l) : 0.0;
  } else {
    // shares of the chosen scores, scaled so that the largest cannot vanish
    const double x = a.score == kSoftmax ? l : (l < 0.0 || l != l ? l : 0.0);
    double mx = live ? x : ninf;
    mx = wave_max_nan_f64(mx);
    double q = live ? exp(x - mx) : 0.0;
    if (a.score == kSigmoid && live) q /= 1.0 + exp(-__builtin_fabs(l));
    const double sum = wave_sum_f64(q);
    w = live ? q / sum : 0.0;
  }
  if (lane < a.k) {
    a.weights[t * a.k + lane] = live ? a.scale * (float)w : 0.0f;
    a.selected[t * a.k + lane] = mine;
    if (a.picked) a.picked[t * a.k + lane] = live ? (float)l : 0.0f;
  }
}

struct RouteBwdArgs {
  const float* dweights;
  const int64_t* selected;
  const float* picked;
  const void* logits;
  int dtype;
  int64_t T, ld;
  int E, k, score, renorm;
  float scale;
  void* dlogits;
};

// One wave per token: the row's gradient in LDS, then written whole.
__global__ __launch_bounds__(256) void moe_route_bwd_kernel(const RouteBwdArgs a) {
  extern __shared__ __align__(16) float row_lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = (int64_t)blockIdx.x * 4 + wave;
  if (t >= a.T) return;
  float* d = row_lds + (int64_t)wave * a.E;
  const float ninf = -__builtin_inff();
  const int64_t sel = lane < a.k ? a.selected[t * a.k + lane] : -1;
  const bool live = sel >= 0 && sel < a.E;
  const float g = live ? a.scale * a.dweights[t * a.k + lane] : 0.0f;
  const float l = live ? a.picked[t * a.k + lane] : ninf;
  float mine = 0.0f;
  const bool dense = a.score == kSoftmax && !a.renorm;
  if (a.renorm) {
    const float x = a.score == kSoftmax ? l : (l < 0.0f || l != l ? l : 0.0f);
    const float mx = (float)wave_max_nan_f64(live ? x : ninf);
    float q = live ? expf(x - mx) : 0.0f;
    const float en = expf(-fabsf(l));
    if (a.score == kSigmoid && live) q /= 1.0f + en;
    const float sum = wave_sum_f32(q);
    const float w = live ? q / sum : 0.0f;
    const float dot = wave_sum_f32(g * w);
    mine = w * (g - dot);
    // 1 - sigmoid(l)
    if (a.score == kSigmoid) mine *= (l > 0.0f ? en : 1.0f) / (1.0f + en);
  } else if (a.score == kSigmoid) {
    const float en = expf(-fabsf(l)), r = 1.0f / (1.0f + en);
    mine = g * en * r * r;
  }
  if (!dense || !__any(live)) {
    for (int e = lane; e < a.E; e += 64) d[e] = 0.0f;
    __builtin_amdgcn_wave_barrier();
    if (live && !dense) d[sel] = mine;
  } else {
    float m = ninf;
    bool bad = false;
    for (int e = lane; e < a.E; e += 64) {
      const float x = load_as_f32(a.logits, a.dtype, t * a.ld + e);
      m = fmaxf(m, x);
      bad |= x != x;
    }
    m = __any(bad) ? __builtin_nanf("") : wave_max(m);
    float z = 0.0f;
    for (int e = lane; e < a.E; e += 64) z += expf(load_as_f32(a.logits, a.dtype, t * a.ld + e) - m);
    z = wave_sum_f32(z);
    const float p = live ? expf(l - m) / z : 0.0f;
    const float dot = wave_sum_f32(g * p);
    for (int e = lane; e < a.E; e += 64) d[e] = -dot * (expf(load_as_f32(a.logits, a.dtype, t * a.ld + e) - m) / z);
    __builtin_amdgcn_wave_barrier();
    if (live) d[sel] += g * p;
  }
  __builtin_amdgcn_wave_barrier();
  for (int e = lane; e < a.E; e += 64) store_f32_as(a.dlogits, a.dtype, t * a.E + e, d[e]);
}

// ---------------------------------------------------------------------------
// Expert order: a stable counting sort of the R = T * k slots by expert, bin E
// holding the slots that name none.  A work-group takes `chunk` consecutive
// slots, wave w of it the w-th sixteenth.
// ---------------------------------------------------------------------------
constexpr int kOrderWaves = 16;
constexpr int kOrderThreads = 64 * kOrderWaves;
constexpr int kOrderBlocks = 256;

// Slots per work-group: a multiple of its threads, at most kOrderBlocks groups.
__host__ __device__ inline int64_t order_chunk(int64_t R) {
  const int64_t c = (R + kOrderBlocks - 1) / kOrderBlocks;
  const int64_t least = c < 4096 ? 4096 : c;
  return (least + kOrderThreads - 1) / kOrderThreads * kOrderThreads;
}

SFP8_DEV int order_bin(const int64_t* sel, int64_t i, int E) {
  const int64_t e = sel[i];
  return e >= 0 && e < E ? (int)e : E;
}

// counts[b][e]: slots of work-group b that name expert e.
__global__ __launch_bounds__(kOrderThreads) void moe_order_count_kernel(const int64_t* __restrict__ sel, int64_t R,
                                                                         int64_t chunk, int E,
                                                                         int* __restrict__ counts) {
  extern __shared__ int hist[];
  for (int e = threadIdx.x; e <= E; e += kOrderThreads) hist[e] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * chunk;
  const int64_t i1 = i0 + chunk < R ? i0 + chunk : R;
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kOrderThreads) atomicAdd(&hist[order_bin(sel, i, E)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e <= E; e += kOrderThreads) counts[(int64_t)blockIdx.x * (E + 1) + e] = hist[e];
}

__global__ __launch_bounds__(kOrderThreads) void moe_order_place_kernel(
    const int64_t* __restrict__ sel, int64_t R, int64_t chunk, int k, int E, const int* __restrict__ counts,
    int64_t* __restrict__ token_index, int64_t* __restrict__ inverse, int* __restrict__ offsets) {
  extern __shared__ int next[];  // [waves][E + 1]: the next row of each bin, per wave
  __shared__ int part[kOrderWaves + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nb = gridDim.x, bins = E + 1;
  for (int e = threadIdx.x; e < kOrderWaves * bins; e += kOrderThreads) next[e] = 0;
  __syncthreads();
  int* mine = next + wave * bins;
  const int64_t per = chunk / kOrderWaves;
  const int64_t i0 = (int64_t)blockIdx.x * chunk + wave * per;
  const int64_t i1 = i0 + per < R ? i0 + per : R;
  for (int64_t i = i0 + lane; i < i1; i += 64) atomicAdd(&mine[order_bin(sel, i, E)], 1);
  __syncthreads();
  // start of each bin: the totals of the bins before it, then this bin's slots of earlier work-groups
  for (int e0 = 0, carry = 0; e0 < bins; e0 += kOrderThreads) {
    const int e = e0 + threadIdx.x;
    int total = 0, before = 0;
    if (e < bins) {
      if (counts) {
        for (int b = 0; b < nb; ++b) {
          const int c = counts[(int64_t)b * bins + e];
          before += b < (int)blockIdx.x ? c : 0;
          total += c;
        }
      } else {
        for (int w = 0; w < kOrderWaves; ++w) total += next[w * bins + e];
      }
    }
    int scan = total;  // inclusive over the wave's bins
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(scan, o, 64);
      scan += lane >= o ? x : 0;
    }
    if (lane == 63) part[wave] = scan;
    __syncthreads();
    int base = carry, all = carry;
    for (int w = 0; w < kOrderWaves; ++w) {
      base += w < wave ? part[w] : 0;
      all += part[w];
    }
    __syncthreads();
    carry = all;
    if (e < bins) {
      if (blockIdx.x == 0 && e < E) offsets[e] = base + scan;
      int at = base + scan - total + before;
      for (int w = 0; w < kOrderWaves; ++w) {
        const int c = next[w * bins + e];
        next[w * bins + e] = at;
        at += c;
      }
    }
  }
  __syncthreads();
  int bits = 0;
  while ((1 << bits) < bins) ++bits;
  for (int64_t i = i0 + lane; i - lane < i1; i += 64) {
    const bool in = i < i1;
    const int e = in ? order_bin(sel, i, E) : 0;
    uint64_t same = __ballot(in);  // the lanes of this step with the same bin
    for (int b = 0; b < bits; ++b) {
      const uint64_t y = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? y : ~y;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    const int row = in ? mine[e] + rank : 0;
    __builtin_amdgcn_wave_barrier();
    if (in && rank == 0) mine[e] = row + __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (in) {
      inverse[i] = e < E ? row : -1;
      token_index[row] = i / k;
    }
  }
}

// ---------------------------------------------------------------------------
// Combine: out[t] = sum over j of w[t, j] rows[inv[t, j]], summed in 32 bits in
// slot order and rounded once; slots whose row is out of range add nothing.
// `lanes` lanes (a power of two) take one token, U elements at a time.
// ---------------------------------------------------------------------------
template <int DT, bool VEC>
struct Unit {  // U consecutive elements as fp32
  static constexpr int U = VEC ? (DT == kF32 ? 4 : 8) : 1;
  float x[U];
  SFP8_DEV void load(const void* p, int64_t i) {
    if constexpr (!VEC) {
      x[0] = load_as_f32(p, DT, i);
    } else if constexpr (DT == kF32) {
      const floatx4 v = *reinterpret_cast<const floatx4*>(reinterpret_cast<const float*>(p) + i);
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = v[q];
    } else {
      const intx4 v = *reinterpret_cast<const intx4*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t lo = (uint32_t)v[q] & 0xffffu, hi = (uint32_t)v[q] >> 16;
        x[2 * q] = DT == kBf16 ? bf16_bits_to_f32(lo) : half_bits_to_f32(lo);
        x[2 * q + 1] = DT == kBf16 ? bf16_bits_to_f32(hi) : half_bits_to_f32(hi);
      }
    }
  }
  SFP8_DEV void store(void* p, int64_t i) const {
    if constexpr (!VEC) {
      store_f32_as(p, DT, i, x[0]);
    } else if constexpr (DT == kF32) {
      *reinterpret_cast<floatx4*>(reinterpret_cast<float*>(p) + i) = floatx4{x[0], x[1], x[2], x[3]};
    } else {
      intx4 o;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        o[q] = (int)(DT == kBf16 ? pack2_bf16(x[2 * q], x[2 * q + 1])
                                 : f32_to_half_bits(x[2 * q]) | f32_to_half_bits(x[2 * q + 1]) << 16);
      *reinterpret_cast<intx4*>(reinterpret_cast<uint16_t*>(p) + i) = o;
    }
  }
};

template <int DT, bool VEC>
__global__ __launch_bounds__(256) void moe_combine_kernel(const void* __restrict__ rows, int64_t R, int64_t D,
                                                          const float* __restrict__ weights,
                                                          const int64_t* __restrict__ inv, int64_t T, int k,
                                                          void* __restrict__ out, int lanes) {
  using X = Unit<DT, VEC>;
  const int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) / lanes;
  if (t >= T) return;
  for (int64_t d = (int64_t)(threadIdx.x & (lanes - 1)) * X::U; d < D; d += (int64_t)lanes * X::U) {
    X acc;
#pragma unroll
    for (int q = 0; q < X::U; ++q) acc.x[q] = 0.0f;
    for (int j = 0; j < k; ++j) {
      const int64_t r = inv[t * k + j];
      if (r < 0 || r >= R) continue;
      const float w = weights[t * k + j];
      X v;
      v.load(rows, r * D + d);
#pragma unroll
      for (int q = 0; q < X::U; ++q) acc.x[q] = __builtin_fmaf(w, v.x[q], acc.x[q]);
    }
    acc.store(out, t * D + d);
  }
}

// drows[inv[t, j]] = w[t, j] dout[t], dw[t, j] = <dout[t], rows[inv[t, j]]>
// (either may be null); rows from offsets[E - 1] on, which no slot names, get
// zeros.  One wave per token.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void moe_combine_bwd_kernel(
    const void* __restrict__ dout, const void* __restrict__ rows, int64_t R, int64_t D,
    const float* __restrict__ weights, const int64_t* __restrict__ inv, int64_t T, int k,
    const int* __restrict__ offsets, int E, void* __restrict__ drows, float* __restrict__ dweights) {
  using X = Unit<DT, VEC>;
  const int lane = threadIdx.x & 63;
  const int64_t gw = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), nw = (int64_t)gridDim.x * 4;
  for (int64_t t = gw; t < T; t += nw) {
    for (int j = 0; j < k; ++j) {
      const int64_t r = inv[t * k + j];
      float dot = 0.0f;
      if (r >= 0 && r < R) {
        const float w = weights[t * k + j];
        for (int64_t d = (int64_t)lane * X::U; d < D; d += 64 * X::U) {
          X g, v;
          g.load(dout, t * D + d);
          if (dweights) {
            v.load(rows, r * D + d);
#pragma unroll
            for (int q = 0; q < X::U; ++q) dot = __builtin_fmaf(g.x[q], v.x[q], dot);
          }
          if (drows) {
#pragma unroll
            for (int q = 0; q < X::U; ++q) g.x[q] *= w;
            g.store(drows, r * D + d);
          }
        }
      }
      if (dweights) {
        dot = wave_sum_f32(dot);
        if (lane == 0) dweights[t * k + j] = dot;
      }
    }
  }
  if (!drows) return;
  int64_t used = offsets[E - 1];
  used = used < 0 ? 0 : used;
  X zero;
#pragma unroll
  for (int q = 0; q < X::U; ++q) zero.x[q] = 0.0f;
  for (int64_t r = used + gw; r < R; r += nw)
    for (int64_t d = (int64_t)lane * X::U; d < D; d += 64 * X::U) zero.store(drows, r * D + d);
}

}  // namespace sfp8

// ============================================================================
// C ABI
// ============================================================================
using namespace sfp8;

namespace {
inline int route_status() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}
inline bool al16(const void* p) { return (((uintptr_t)p) & 15u) == 0; }
inline bool bad_dtype(int d) { return d != kF32 && d != kBf16 && d != kF16; }
constexpr int64_t kMaxTokens = (int64_t)1 << 25;  // 64 lanes a token: a launch's work-items stay below 2^32

// dynamic LDS above 64 KiB must be opted into per kernel
template <typename K>
int route_allow_lds(K kernel, size_t bytes) {
  if (bytes <= 65536) return kOk;
  const hipError_t e =
      hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  return e == hipSuccess ? kOk : (int)e;
}

// Calls f<dtype, whole 16-byte units>.
template <template <int, bool> class F, typename... A>
void by_type(int dtype, bool vec, A... args) {
  if (dtype == kF32) vec ? F<kF32, true>::run(args...) : F<kF32, false>::run(args...);
  else if (dtype == kBf16) vec ? F<kBf16, true>::run(args...) : F<kBf16, false>::run(args...);
  else vec ? F<kF16, true>::run(args...) : F<kF16, false>::run(args...);
}

template <int DT, bool VEC>
struct Combine {
  static void run(const void* rows, int64_t R, int64_t D, const float* w, const int64_t* inv, int64_t T, int k,
                  void* out, hipStream_t st) {
    int lanes = 64;
    while (lanes > 1 && (int64_t)(lanes / 2) * Unit<DT, VEC>::U >= D) lanes /= 2;
    const int64_t per = 256 / lanes;
    hipLaunchKernelGGL((moe_combine_kernel<DT, VEC>), dim3((unsigned)((T + per - 1) / per)), dim3(256), 0, st, rows, R,
                       D, w, inv, T, k, out, lanes);
  }
};

template <int DT, bool VEC>
struct CombineBwd {
  static void run(const void* dout, const void* rows, int64_t R, int64_t D, const float* w, const int64_t* inv,
                  int64_t T, int k, const int* offsets, int E, void* drows, float* dw, hipStream_t st) {
    const int64_t nb = (T + 3) / 4;
    hipLaunchKernelGGL((moe_combine_bwd_kernel<DT, VEC>), dim3((unsigned)(nb < 1 ? 1 : nb)), dim3(256), 0, st, dout,
                       rows, R, D, w, inv, T, k, offsets, E, drows, dw);
  }
};
}  // namespace

extern "C" {

int sfp8_moe_route(const void* logits, int dtype, int64_t T, int64_t E, int64_t ld, const float* bias,
                   const void* mask, int score, int64_t groups, int64_t top_groups, int64_t group_best, int64_t top_k,
                   int renorm, float scale, float* weights, int64_t* selected, float* picked, void* stream) {
  if (T > 0 && (!logits || !weights || !selected)) return kErrNullPointer;
  if (T < 0 || T > kMaxTokens || E <= 0 || E > kRouteMaxExperts || ld < 0 || bad_dtype(dtype)) return kErrBadShape;
  if ((score != kSoftmax && score != kSigmoid) || groups <= 0 || groups > 64 || E % groups || top_groups <= 0 ||
      top_groups > groups || (group_best != 1 && group_best != 2))
    return kErrBadShape;
  if (top_k <= 0 || top_k > kRouteMaxK || top_k > top_groups * (E / groups)) return kErrBadShape;
  if (T == 0) return kOk;
  const RouteArgs a{logits, dtype, T, ld, (int)E, (int)top_k, score, (int)groups, (int)top_groups, (int)group_best,
                    renorm, scale, bias, (const uint8_t*)mask, weights, selected, picked};
  hipLaunchKernelGGL(moe_route_kernel, dim3((unsigned)((T + 3) / 4)), dim3(256), 4 * (size_t)E * 8,
                     (hipStream_t)stream, a);
  return route_status();
}

int sfp8_moe_route_bwd(const float* dweights, const int64_t* selected, const float* picked, const void* logits,
                       int dtype, int64_t T, int64_t E, int64_t ld, int score, int64_t top_k, int renorm, float scale,
                       void* dlogits, void* stream) {
  const bool dense = score == kSoftmax && !renorm;
  if (T > 0 && (!dweights || !selected || !picked || !dlogits || (dense && !logits))) return kErrNullPointer;
  if (T < 0 || T > kMaxTokens || E <= 0 || E > kRouteMaxExperts || ld < 0 || bad_dtype(dtype)) return kErrBadShape;
  if ((score != kSoftmax && score != kSigmoid) || top_k <= 0 || top_k > kRouteMaxK || top_k > E) return kErrBadShape;
  if (T == 0) return kOk;
  const RouteBwdArgs a{dweights, selected, picked, logits, dtype, T, ld, (int)E, (int)top_k, score, renorm, scale,
                       dlogits};
  hipLaunchKernelGGL(moe_route_bwd_kernel, dim3((unsigned)((T + 3) / 4)), dim3(256), 4 * (size_t)E * 4,
                     (hipStream_t)stream, a);
  return route_status();
}

int64_t sfp8_moe_expert_order_workspace_ints(int64_t R, int64_t E) {
  if (R < 0 || R > (int64_t)1 << 30 || E <= 0 || E > kRouteMaxExperts) return -1;
  const int64_t chunk = order_chunk(R), nb = (R + chunk - 1) / chunk;
  return nb > 1 ? nb * (E + 1) : 0;
}

int sfp8_moe_expert_order(const int64_t* selected, int64_t R, int64_t top_k, int64_t E, int64_t* token_index,
                          int64_t* inverse, int* offsets, int* ws, int64_t ws_ints, void* stream) {
  if (!offsets || (R > 0 && (!selected || !token_index || !inverse))) return kErrNullPointer;
  const int64_t need = sfp8_moe_expert_order_workspace_ints(R, E);
  if (need < 0 || top_k <= 0 || R % top_k) return kErrBadShape;
  if (need > 0 && (!ws || ws_ints < need)) return kErrWorkspaceTooSmall;
  const int64_t chunk = order_chunk(R);
  const int64_t nb = R > chunk ? (R + chunk - 1) / chunk : 1;
  const size_t lds = (size_t)kOrderWaves * (E + 1) * 4;
  if (const int rc = route_allow_lds(moe_order_place_kernel, lds)) return rc;
  if (nb > 1)
    hipLaunchKernelGGL(moe_order_count_kernel, dim3((unsigned)nb), dim3(kOrderThreads), (size_t)(E + 1) * 4,
                       (hipStream_t)stream, selected, R, chunk, (int)E, ws);
  hipLaunchKernelGGL(moe_order_place_kernel, dim3((unsigned)nb), dim3(kOrderThreads), lds, (hipStream_t)stream,
                     selected, R, chunk, (int)top_k, (int)E, nb > 1 ? ws : nullptr, token_index, inverse, offsets);
  return route_status();
}

int sfp8_moe_combine(const void* rows, int dtype, int64_t R, int64_t D, const float* weights, const int64_t* inverse,
                     int64_t T, int64_t top_k, void* out, void* stream) {
  if ((T > 0 && (!out || !weights || !inverse)) || (R > 0 && T > 0 && !rows)) return kErrNullPointer;
  if (R < 0 || T < 0 || T > kMaxTokens || D <= 0 || top_k <= 0 || top_k > kRouteMaxK || bad_dtype(dtype))
    return kErrBadShape;
  if (T == 0) return kOk;
  const bool vec = D % (dtype == kF32 ? 4 : 8) == 0 && al16(rows) && al16(out);
  by_type<Combine>(dtype, vec, rows, R, D, weights, inverse, T, (int)top_k, out, (hipStream_t)stream);
  return route_status();
}

int sfp8_moe_combine_bwd(const void* dout, const void* rows, int dtype, int64_t R, int64_t D, const float* weights,
                         const int64_t* inverse, int64_t T, int64_t top_k, const int* offsets, int64_t E, void* drows,
                         float* dweights, void* stream) {
  if ((T > 0 && (!dout || !weights || !inverse)) || (R > 0 && dweights && T > 0 && !rows) || (drows && !offsets))
    return kErrNullPointer;
  if (R < 0 || T < 0 || T > kMaxTokens || D <= 0 || top_k <= 0 || top_k > kRouteMaxK || bad_dtype(dtype) || E <= 0)
    return kErrBadShape;
  if ((T == 0 && R == 0) || (!drows && !dweights)) return kOk;
  const bool vec = D % (dtype == kF32 ? 4 : 8) == 0 && al16(rows) && al16(dout) && al16(drows);
  by_type<CombineBwd>(dtype, vec, dout, rows, R, D, weights, inverse, T, (int)top_k, offsets, (int)E, drows, dweights,
                      (hipStream_t)stream);
  return route_status();
}

}  // extern "C"
