// The global norm of many gradients and their scaling to a largest norm
// (gfx950): what a training step does between the backward pass and the
// optimizer's momentum stage (optim.hip).
//
//   n = sqrt(sum over all tensors and elements of g^2)
//   c = min(1, max_norm / (n + 1e-6)),  out = round(c * g)
//
// The squares are summed in 64 bits (a square of a 32-bit number cannot
// overflow there, and 64-bit FMAs cost a few percent of the time the bytes
// take), in an order that depends on the sizes and types alone, not on the
// addresses: every work-group sums its own chunks, each thread the same elements
// of them, then the sums are added in order.  Bound by HBM: each
// gradient is read once for the norm and, where c != 1 or the result goes
// elsewhere, read again and written.
#include "common.h"

#include <type_traits>

namespace sfp8 {

enum : int { kF32 = 0, kBf16 = 1, kF16 = 2 };

// The tensors of one launch, passed by value: 4 KiB of kernel arguments.
constexpr int kClipTensors = 120;
constexpr int kClipChunk = 65536;   // bytes of a gradient that one work-group takes at a time
constexpr int kClipBlocks = 2048;   // work-groups of a launch, at most
constexpr int kClipThreads = 256;
constexpr int64_t kClipLastLevelCache = (int64_t)256 << 20;
constexpr int kClipUnroll = 8;      // 16-byte loads of a thread in flight

struct ClipTable {
  const void* in[kClipTensors];
  void* out[kClipTensors];
  int64_t n[kClipTensors];
  uint32_t first[kClipTensors + 1];  // first chunk of each tensor; [count]: all chunks
  uint8_t dtype[kClipTensors];
  int count;
  bool in_place;  // every out[i] == in[i]
};

SFP8_DEV float half_to_f32(uint32_t b) { return (float)__builtin_bit_cast(_Float16, (uint16_t)b); }

// Finds the tensor of a chunk: the largest i with first[i] <= c.  The lanes hold
// the whole list, so that a chunk takes no loads that wait for each other.
struct ClipFinder {
  uint32_t f0, f1;
  SFP8_DEV explicit ClipFinder(const ClipTable& tab) {
    const int lane = threadIdx.x & 63;
    f0 = lane < tab.count ? tab.first[lane] : ~0u;
    f1 = lane + 64 < tab.count ? tab.first[lane + 64] : ~0u;
  }
  SFP8_DEV int operator()(uint32_t c) const {
    return __popcll(__ballot(f0 <= c)) + __popcll(__ballot(f1 <= c)) - 1;
  }
};

// Elements 0 .. U - 1 of 16 bytes as fp32.
template <int DT>
struct Pack {
  static constexpr int U = DT == kF32 ? 4 : 8;
  static constexpr int kSize = DT == kF32 ? 4 : 2;
  SFP8_DEV static float get(const intx4& v, int i) {
    if (DT == kF32) return __uint_as_float((uint32_t)v[i]);
    const uint32_t b = ((uint32_t)v[i >> 1] >> (16 * (i & 1))) & 0xffffu;
    return DT == kBf16 ? bf16_bits_to_f32(b) : half_to_f32(b);
  }
  SFP8_DEV static float load(const void* p, int64_t i) {
    if (DT == kF32) return reinterpret_cast<const float*>(p)[i];
    const uint32_t b = reinterpret_cast<const uint16_t*>(p)[i];
    return DT == kBf16 ? bf16_bits_to_f32(b) : half_to_f32(b);
  }
  SFP8_DEV static uint32_t bits(float f) {
    if (DT == kF32) return __float_as_uint(f);
    return DT == kBf16 ? f32_to_bf16_bits(f) : (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f);
  }
  SFP8_DEV static void store(void* p, int64_t i, float f) {
    if (DT == kF32) reinterpret_cast<float*>(p)[i] = f;
    else reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)bits(f);
  }
  SFP8_DEV static intx4 scaled(const intx4& v, float c) {
    intx4 o;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (DT == kF32) o[q] = (int)bits(get(v, q) * c);
      else o[q] = (int)(bits(get(v, 2 * q) * c) | bits(get(v, 2 * q + 1) * c) << 16);
    }
    return o;
  }
};

// 16 bytes at any element's address: global memory takes them there in one access.
typedef int intx4_any __attribute__((ext_vector_type(4), aligned(2)));

// The elements [e0, e1) of a chunk: those before the first 16-byte boundary,
// whole 16-byte vectors, and the rest.  one(i) takes element i, vec(i, v) the
// vector v that starts at element i.  ONCE: loads that pass the caches by.  ANY:
// vectors from e0 on, wherever that lies in its 16 bytes.
template <int DT, bool ONCE, bool ANY, typename One, typename Vec>
SFP8_DEV void clip_walk(const void* p, int64_t e0, int64_t e1, One one, Vec vec) {
  using P = Pack<DT>;
  using V = std::conditional_t<ANY, intx4_any, intx4>;
  constexpr int kStep = kClipThreads * P::U;
  const char* at = reinterpret_cast<const char*>(p) + e0 * P::kSize;
  const int n = (int)(e1 - e0);
  const int lead = ANY ? 0 : (int)((16 - ((uintptr_t)at & 15)) & 15) / P::kSize;
  const int v0 = lead < n ? lead : n, v1 = v0 + (n - v0) / P::U * P::U;
  if ((int)threadIdx.x < v0) one(e0 + threadIdx.x);
  int i = v0 + (int)threadIdx.x * P::U;
  for (; i + (kClipUnroll - 1) * kStep < v1; i += kClipUnroll * kStep) {  // kClipUnroll loads in flight
    intx4 v[kClipUnroll];
#pragma unroll
    for (int q = 0; q < kClipUnroll; ++q) {
      const V* x = reinterpret_cast<const V*>(at + (i + q * kStep) * P::kSize);
      v[q] = ONCE ? __builtin_nontemporal_load(x) : *x;
    }
#pragma unroll
    for (int q = 0; q < kClipUnroll; ++q) vec(e0 + i + q * kStep, v[q]);
  }
  for (; i < v1; i += kStep) {
    const intx4 v = *reinterpret_cast<const V*>(at + i * P::kSize);
    vec(e0 + i, v);
  }
  if (v1 + (int)threadIdx.x < n) one(e0 + v1 + threadIdx.x);
}

template <int DT, bool ONCE>
SFP8_DEV double clip_squares(const void* p, int64_t e0, int64_t e1) {
  using P = Pack<DT>;
  double s = 0.0;
  clip_walk<DT, ONCE, true>(
      p, e0, e1,
      [&](int64_t i) {
        const double x = P::load(p, i);
        s = __builtin_fma(x, x, s);
      },
      [&](int64_t, const intx4& v) {
#pragma unroll
        for (int q = 0; q < P::U; ++q) {
          const double x = P::get(v, q);
          s = __builtin_fma(x, x, s);
        }
      });
  return s;
}

template <int DT, bool ONCE>
SFP8_DEV void clip_scale(const void* p, void* o, int64_t e0, int64_t e1, float c, bool aligned) {
  using P = Pack<DT>;
  const auto one = [&](int64_t i) { P::store(o, i, P::load(p, i) * c); };
  if (!aligned) {  // in and out sit differently in their 16 bytes
    for (int64_t i = e0 + threadIdx.x; i < e1; i += kClipThreads) one(i);
    return;
  }
  clip_walk<DT, ONCE, false>(p, e0, e1, one, [&](int64_t i, const intx4& v) {
    __builtin_nontemporal_store(P::scaled(v, c), reinterpret_cast<intx4*>(reinterpret_cast<char*>(o) + i * P::kSize));
  });
}

// part[blockIdx.x] = the squares of this work-group's chunks.
template <bool ONCE>
__global__ __launch_bounds__(kClipThreads) void clip_norm_kernel(const ClipTable tab, double* __restrict__ part) {
  __shared__ double red[kClipThreads / 64];
  const ClipFinder find(tab);
  const uint32_t chunks = tab.first[tab.count];
  double s = 0.0;
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = find(c);
    const int dt = tab.dtype[i];
    const int64_t per = kClipChunk / (dt == kF32 ? 4 : 2);
    const int64_t e0 = (int64_t)(c - tab.first[i]) * per;
    const int64_t e1 = e0 + per < tab.n[i] ? e0 + per : tab.n[i];
    s += dt == kF32 ? clip_squares<kF32, ONCE>(tab.in[i], e0, e1)
                    : dt == kBf16 ? clip_squares<kBf16, ONCE>(tab.in[i], e0, e1)
                                  : clip_squares<kF16, ONCE>(tab.in[i], e0, e1);
  }
  s = wave_sum_f64(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// The norm from the partial sums, the same in every work-group that asks.
SFP8_DEV float clip_norm_of(const double* part, int parts) {
  __shared__ double red[kClipThreads / 64];
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += kClipThreads) s += part[i];
  s = wave_sum_f64(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  return (float)sqrt((red[0] + red[1]) + (red[2] + red[3]));
}

__global__ __launch_bounds__(kClipThreads) void clip_norm_out_kernel(const double* __restrict__ part, int parts,
                                                                     float* __restrict__ norm) {
  const float n = clip_norm_of(part, parts);
  if (threadIdx.x == 0) *norm = n;
}

template <bool ONCE>
__global__ __launch_bounds__(kClipThreads) void clip_scale_kernel(const ClipTable tab, const double* __restrict__ part,
                                                                  int parts, float max_norm, bool backwards,
                                                                  float* __restrict__ norm) {
  const float n = clip_norm_of(part, parts);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
  float f = max_norm / (n + 1e-6f);
  f = f > 1.0f ? 1.0f : f;  // keeps NaN
  if (f == 1.0f && tab.in_place) return;  // x * 1 is x
  const ClipFinder find(tab);
  const uint32_t chunks = tab.first[tab.count];
  for (uint32_t b = blockIdx.x; b < chunks; b += gridDim.x) {
    const uint32_t c = backwards ? chunks - 1 - b : b;
    const int i = find(c);
    if (f == 1.0f && tab.in[i] == tab.out[i]) continue;
    const int dt = tab.dtype[i];
    const int64_t per = kClipChunk / (dt == kF32 ? 4 : 2);
    const int64_t e0 = (int64_t)(c - tab.first[i]) * per;
    const int64_t e1 = e0 + per < tab.n[i] ? e0 + per : tab.n[i];
    const bool aligned = (((uintptr_t)tab.in[i] ^ (uintptr_t)tab.out[i]) & 15u) == 0;
    if (dt == kF32) clip_scale<kF32, ONCE>(tab.in[i], tab.out[i], e0, e1, f, aligned);
    else if (dt == kBf16) clip_scale<kBf16, ONCE>(tab.in[i], tab.out[i], e0, e1, f, aligned);
    else clip_scale<kF16, ONCE>(tab.in[i], tab.out[i], e0, e1, f, aligned);
  }
}

}  // namespace sfp8

// ============================================================================
// C ABI
// ============================================================================
using namespace sfp8;

namespace {
inline int clip_status() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}
inline int64_t clip_chunks(int64_t n, int dtype) {
  const int64_t bytes = n * (dtype == kF32 ? 4 : 2);
  return (bytes + kClipChunk - 1) / kClipChunk;
}

// Tables of up to kClipTensors tensors each (tensors without elements are left
// out): f(table, work-groups).
template <typename F>
void clip_tables(int64_t count, const void* const* in, void* const* out, const int64_t* n, const int* dtype, F f) {
  ClipTable tab;
  tab.count = 0;
  tab.first[0] = 0;
  tab.in_place = true;
  const auto flush = [&] {
    if (tab.count == 0) return;
    const uint32_t chunks = tab.first[tab.count];
    f(tab, (int)(chunks < (uint32_t)kClipBlocks ? chunks : (uint32_t)kClipBlocks));
    tab.count = 0;
    tab.in_place = true;
  };
  for (int64_t i = 0; i < count; ++i) {
    if (n[i] == 0) continue;
    const int64_t c = clip_chunks(n[i], dtype[i]);
    if (tab.count == kClipTensors || (tab.count && tab.first[tab.count] + c > 0x7fffffff)) flush();
    const int j = tab.count++;
    tab.in[j] = in[i];
    tab.out[j] = out ? out[i] : nullptr;
    tab.in_place &= tab.out[j] == tab.in[j];
    tab.n[j] = n[i];
    tab.dtype[j] = (uint8_t)dtype[i];
    tab.first[j + 1] = (j ? tab.first[j] : 0) + (uint32_t)c;
  }
  flush();
}

int clip_check(int64_t count, const void* const* in, const int64_t* n, const int* dtype) {
  if (count < 0) return kErrBadShape;
  if (count > 0 && (!in || !n || !dtype)) return kErrNullPointer;
  for (int64_t i = 0; i < count; ++i) {
    if (n[i] < 0 || n[i] > (int64_t)1 << 40 || dtype[i] < 0 || dtype[i] > 2) return kErrBadShape;
    if (n[i] > 0 && !in[i]) return kErrNullPointer;
    if ((uintptr_t)in[i] % (dtype[i] == kF32 ? 4 : 2)) return kErrBadAlignment;
  }
  return kOk;
}
}  // namespace

extern "C" {

int64_t sfp8_grad_norm_workspace_doubles(int64_t count) {
  return count < 0 ? -1 : (count + kClipTensors - 1) / kClipTensors * kClipBlocks + kClipBlocks;
}

int sfp8_grad_norm(int64_t count, const void* const* grads, const int64_t* n, const int* dtype, float* norm,
                   double* ws, int64_t ws_doubles, void* stream) {
  if (const int rc = clip_check(count, grads, n, dtype)) return rc;
  if (!norm || !ws) return kErrNullPointer;
  if (ws_doubles < sfp8_grad_norm_workspace_doubles(count)) return kErrWorkspaceTooSmall;
  hipStream_t st = (hipStream_t)stream;
  int parts = 0;
  clip_tables(count, grads, nullptr, n, dtype, [&](const ClipTable& tab, int blocks) {
    hipLaunchKernelGGL(clip_norm_kernel<true>, dim3(blocks), dim3(kClipThreads), 0, st, tab, ws + parts);
    parts += blocks;
  });
  hipLaunchKernelGGL(clip_norm_out_kernel, dim3(1), dim3(kClipThreads), 0, st, ws, parts, norm);
  return clip_status();
}

int sfp8_grad_clip(int64_t count, const void* const* grads, void* const* out, const int64_t* n, const int* dtype,
                   float max_norm, float* norm, double* ws, int64_t ws_doubles, void* stream) {
  if (const int rc = clip_check(count, grads, n, dtype)) return rc;
  if (!norm || !ws || (count > 0 && !out)) return kErrNullPointer;
  if (!(max_norm >= 0.0f)) return kErrBadShape;
  for (int64_t i = 0; i < count; ++i) {
    if (n[i] > 0 && !out[i]) return kErrNullPointer;
    if ((uintptr_t)out[i] % (dtype[i] == kF32 ? 4 : 2)) return kErrBadAlignment;
  }
  if (ws_doubles < sfp8_grad_norm_workspace_doubles(count)) return kErrWorkspaceTooSmall;
  hipStream_t st = (hipStream_t)stream;
  int64_t bytes = 0;
  bool elsewhere = false;
  for (int64_t i = 0; i < count; ++i) {
    bytes += n[i] * (dtype[i] == kF32 ? 4 : 2);
    elsewhere |= n[i] > 0 && out[i] != grads[i];
  }
  // Which loads pass the caches by, and which way the second pass goes.  us of
  // 63 / 151 / 1208 MB, below the limit, scaled in place, scaled elsewhere:
  //   neither, the second backwards   16 31 211 | 34 75 677 | 34 73 655
  //   both, backwards                 13 29 183 | 38 83 643 | 36 80 634
  //   the norm's, forwards            13 30 183 | 35 73 647 | 35 80 666
  const bool large = bytes > kClipLastLevelCache;
  const bool norm_once = !elsewhere || large, scale_once = elsewhere && large;
  int parts = 0;
  clip_tables(count, grads, out, n, dtype, [&](const ClipTable& tab, int blocks) {
    if (norm_once) hipLaunchKernelGGL(clip_norm_kernel<true>, dim3(blocks), dim3(kClipThreads), 0, st, tab, ws + parts);
    else hipLaunchKernelGGL(clip_norm_kernel<false>, dim3(blocks), dim3(kClipThreads), 0, st, tab, ws + parts);
    parts += blocks;
  });
  if (parts == 0) {  // nothing to scale: the norm is 0
    hipLaunchKernelGGL(clip_norm_out_kernel, dim3(1), dim3(kClipThreads), 0, st, ws, 0, norm);
    return clip_status();
  }
  float* first = norm;
  clip_tables(count, grads, out, n, dtype, [&](const ClipTable& tab, int blocks) {
    if (scale_once)
      hipLaunchKernelGGL(clip_scale_kernel<true>, dim3(blocks), dim3(kClipThreads), 0, st, tab, ws, parts, max_norm,
                         elsewhere, first);
    else
      hipLaunchKernelGGL(clip_scale_kernel<false>, dim3(blocks), dim3(kClipThreads), 0, st, tab, ws, parts, max_norm,
                         elsewhere, first);
    first = nullptr;
  });
  return clip_status();
}

}  // extern "C"
