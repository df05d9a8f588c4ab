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

// 16 and 8 bytes at any element's address: global memory takes them there in
// one access.
typedef int intx4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef int intx2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef float floatx4_any __attribute__((ext_vector_type(4), aligned(4)));

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

// ---------------------------------------------------------------------------
// Reductions over the L lanes of a token (L a power of two, its lanes aligned
// to L).  share<S>(x) gives two values whose combination is that of x with the
// lane S away, where the S lanes below already agree: DPP within 16 lanes
// (quad permutes, mirrors of half rows and rows), the lane swaps beyond.
// ---------------------------------------------------------------------------
struct Two {
  uint32_t a, b;
};
template <int S>
SFP8_DEV Two share(uint32_t x) {
  static_assert(S == 1 || S == 2 || S == 4 || S == 8 || S == 16 || S == 32, "");
  if constexpr (S == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return {r[0], r[1]};
  } else if constexpr (S == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return {r[0], r[1]};
  } else {
    constexpr int ctrl = S == 1 ? 0xB1 : S == 2 ? 0x4E : S == 4 ? 0x141 : 0x140;
    return {x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, ctrl, 0xf, 0xf, true)};
  }
}
template <int S>
SFP8_DEV void share_f(float x, float& a, float& b) {
  const Two t = share<S>(__float_as_uint(x));
  a = __uint_as_float(t.a);
  b = __uint_as_float(t.b);
}
template <int L, int S = 1, class F>
SFP8_DEV float reduce_f(float x, F f) {
  if constexpr (S < L) {
    float a, b;
    share_f<S>(x, a, b);
    return reduce_f<L, S * 2>(f(a, b), f);
  } else {
    return x;
  }
}
template <int L, int S = 1>
SFP8_DEV uint32_t reduce_max_u(uint32_t x) {
  if constexpr (S < L) {
    const Two t = share<S>(x);
    return reduce_max_u<L, S * 2>(t.a > t.b ? t.a : t.b);
  } else {
    return x;
  }
}
template <int L>
SFP8_DEV float lanes_max(float x) {
  return reduce_f<L>(x, [](float a, float b) { return fmaxf(a, b); });
}
template <int L>
SFP8_DEV float lanes_min(float x) {
  return reduce_f<L>(x, [](float a, float b) { return fminf(a, b); });
}
template <int L>
SFP8_DEV float lanes_sum(float x) {
  return reduce_f<L>(x, [](float a, float b) { return a + b; });
}

constexpr float kLog2E = 1.4426950408889634f;
SFP8_DEV float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * kLog2E); }

// How the experts of a token lie in its L lanes: each group (all of them, when
// there are none) has the G lanes g * G .. g * G + G - 1 of group g, and lane
// `sub` of them holds, in chunks of four, members 4 * (c * G + sub) + i.
struct RouteLayout {
  int G, gs;  // lanes and members of a group
  int g, sub;
  SFP8_DEV int member(int c) const { return 4 * (c * G + sub); }
};

// Four values of a row, from element `at` of p on.
SFP8_DEV void load4(float (&x)[4], const void* p, int dtype, int64_t at) {
  if (dtype == kF32) {
    const floatx4_any v = *reinterpret_cast<const floatx4_any*>(reinterpret_cast<const float*>(p) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = v[i];
  } else {
    const intx2_any v = *reinterpret_cast<const intx2_any*>(reinterpret_cast<const uint16_t*>(p) + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t b = ((uint32_t)v[i >> 1] >> (16 * (i & 1))) & 0xffffu;
      x[i] = dtype == kBf16 ? bf16_bits_to_f32(b) : half_bits_to_f32(b);
    }
  }
}

// The V logits of a lane: those past the group's members, and all where `on` is
// false, read as -inf.  at: the group's first logit.
template <int V>
SFP8_DEV void load_logits(float (&l)[V], const void* p, int dtype, int64_t at, const RouteLayout& lay, bool on) {
  const float ninf = -__builtin_inff();
  if (lay.gs == lay.G * V && __all(on)) {  // nothing to leave out
    if (dtype == kF32) {  // uniform, once: the loads go out together
#pragma unroll
      for (int c = 0; c < V / 4; ++c) load4(*reinterpret_cast<float(*)[4]>(l + 4 * c), p, kF32, at + lay.member(c));
    } else if (dtype == kBf16) {
#pragma unroll
      for (int c = 0; c < V / 4; ++c) load4(*reinterpret_cast<float(*)[4]>(l + 4 * c), p, kBf16, at + lay.member(c));
    } else {
#pragma unroll
      for (int c = 0; c < V / 4; ++c) load4(*reinterpret_cast<float(*)[4]>(l + 4 * c), p, kF16, at + lay.member(c));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) l[j] = ninf;
  if (!on) return;
#pragma unroll
  for (int c = 0; c < V / 4; ++c) {
    const int m = lay.member(c);
    if (m + 4 <= lay.gs) {
      load4(*reinterpret_cast<float(*)[4]>(l + 4 * c), p, dtype, at + m);
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (m + i < lay.gs) l[4 * c + i] = load_as_f32(p, dtype, at + m + i);
    }
  }
}

// A double as an integer in the order of ranks_above: NaN is all ones, -inf
// (what cannot be taken) is 0.
SFP8_DEV uint64_t rank_bits(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
  const uint64_t ord = b >> 63 ? ~b : b | 1ull << 63;
  return x != x ? ~0ull : x == -__builtin_inf() ? 0ull : ord;
}
template <int S = 1>
SFP8_DEV uint64_t wave_max_u64(uint64_t x) {
  if constexpr (S < 64) {
    const Two lo = share<S>((uint32_t)x), hi = share<S>((uint32_t)(x >> 32));
    const uint64_t a = (uint64_t)hi.a << 32 | lo.a, b = (uint64_t)hi.b << 32 | lo.b;
    return wave_max_u64<S * 2>(a > b ? a : b);
  } else {
    return x;
  }
}

// ---------------------------------------------------------------------------
// The selection by the definition, in 64 bits, of one token by a whole wave:
// for rows that hold NaN or +inf and for those whose order 32 bits do not
// settle.  Returns the expert of slot `lane`, or -1.  v[e] (LDS) is the order
// value of expert e as rank_bits, 0 where it cannot be taken (any more); the
// row's logits follow it.  The code is seldom run and so comes from memory: its
// length counts for more than its steps, hence one exponential, one quotient
// and few unrolled loops.
// ---------------------------------------------------------------------------
SFP8_DEV int route_exact(const RouteArgs& a, int64_t t, uint64_t* v) {
  const int lane = threadIdx.x & 63;
  const double ninf = -__builtin_inf();
  const int64_t row = t * a.ld;
  const bool softmax = a.score == kSoftmax;
  const bool two_best = a.groups > 1 && a.group_best == 2;
  float* l = reinterpret_cast<float*>(v + a.E);  // the row
  double m = ninf;
#pragma unroll 1
  for (int e0 = lane; e0 < a.E; e0 += 256) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = e0 + 64 * i < a.E ? load_as_f32(a.logits, a.dtype, row + e0 + 64 * i) : -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (e0 + 64 * i < a.E) l[e0 + 64 * i] = x[i];
      m = ranks_above(x[i], m) ? (double)x[i] : m;
    }
  }
  const bool scores = a.bias || two_best;
  if (scores) {  // which d holds until they are ranked
    m = wave_max_nan_f64(m);
    double z = 0.0;
    double* d = reinterpret_cast<double*>(v);
#pragma unroll 1
    for (int e = lane; e < a.E; e += 64) {
      const double x = exp(softmax ? l[e] - m : -(double)l[e]);
      z += x;
      d[e] = x;
    }
    z = wave_sum_f64(z);
#pragma unroll 1
    for (int e = lane; e < a.E; e += 64) {
      const double x = (softmax ? d[e] : 1.0) / (softmax ? z : 1.0 + d[e]);
      v[e] = l[e] == -__builtin_inff() ? 0ull : rank_bits(a.bias ? x + (double)a.bias[e] : x);
    }
  } else {
#pragma unroll 1
    for (int e = lane; e < a.E; e += 64) v[e] = rank_bits(l[e]);
  }
  __builtin_amdgcn_wave_barrier();
  if (a.groups > 1) {
    const int gs = a.E / a.groups;
    uint64_t b1 = 0, b2 = 0;  // the best two of group `lane`
    if (lane < a.groups) {
#pragma unroll 1
      for (int e0 = 0; e0 < gs; e0 += 4) {
        uint64_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = e0 + i < gs ? v[lane * gs + e0 + i] : 0ull;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          b2 = x[i] > b1 ? b1 : x[i] > b2 ? x[i] : b2;
          b1 = x[i] > b1 ? x[i] : b1;
        }
      }
    }
    uint64_t g = b1;
    if (two_best && b2) {
      const auto value = [](uint64_t x) {
        return x == ~0ull ? __builtin_nan("") : __builtin_bit_cast(double, x >> 63 ? x & ~(1ull << 63) : ~x);
      };
      g = rank_bits(value(b1) + value(b2));
    }
    int rank = 0;
#pragma unroll 1
    for (int j = 0; j < a.groups; ++j) {
      const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(g >> 32), j) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)g, j);
      rank += o > g || (o == g && j < lane);
    }
    const uint64_t keep = __ballot(lane < a.groups && g && rank < a.top_groups);
    __builtin_amdgcn_wave_barrier();
    const bool again = two_best && !a.bias;  // the order is that of the logits
#pragma unroll 1
    for (int e = lane; e < a.E; e += 64) v[e] = keep >> (e / gs) & 1 ? (again ? rank_bits(l[e]) : v[e]) : 0ull;
    __builtin_amdgcn_wave_barrier();
  }
  int mine = -1;
#pragma unroll 1
  for (int s = 0; s < a.k; ++s) {
    uint64_t best = 0;
    int at = a.E;
#pragma unroll 1
    for (int e0 = lane; e0 < a.E; e0 += 256) {
      uint64_t x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = e0 + 64 * i < a.E ? v[e0 + 64 * i] : 0ull;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        at = x[i] > best ? e0 + 64 * i : at;
        best = x[i] > best ? x[i] : best;
      }
    }
    const uint64_t m = wave_max_u64(best);
    if (m == 0) break;
    // the lowest index of them
    at = a.E - (int)reduce_max_u<64>(best == m ? (uint32_t)(a.E - at) : 0u);
    mine = lane == s ? at : mine;
    if (lane == 0) v[at] = 0ull;
    __builtin_amdgcn_wave_barrier();
  }
  return mine;
}

// ---------------------------------------------------------------------------
// Routing, L lanes a token, V values a lane, 64 / L tokens a wave.
//
// The order.  Each expert gets a key of 31 bits, a rank of 21 to 23 bits above
// its inverted index, so that keys differ and the larger key comes first.
// 16-bit logits without a bias have the order of their own bits as the rank.
// Others are put on a fixed-point scale between a low value and the row's
// largest: rank = 1 + (value - low) * scale, with the mantissa of a number
// from 2^23 on as the integer; what is below low has rank 0 and is not taken.  Each
// step to it keeps the order, so ranks that differ are in the order of the
// 32-bit values.  Without groups and with more lanes than slots the low value
// is the smallest of the lanes' largest, less the errors of biased scores: L
// values are no smaller, so the top_k + 1 first are among them.  The next key
// below `top` is max(key - top) + top in wrapping arithmetic (keys below top wrap
// to 2^31 and above, those from top on stay below), a subtraction and half a max3
// for each value and log2(L) lane steps, with nothing to clear.
//
// Its limits.  Where two neighbours of the top_k + 1 first are closer than
// their errors, the first few are put in order again by their values in 64 bits,
// and so are the groups where two are that close at the border of those kept.
// Where more than four experts behind the last are that close, or for a biased
// softmax, whose sum is over the whole row, the whole selection is done again by
// the definition in 64 bits (route_exact), as it is for rows with NaN or +inf.
// Without a bias that takes two logits that differ on one step of the
// scale (equal ones are in the order of their indices): about 1 of 10^4 tokens
// at 256 normal logits.  With one, scores are off.  An exponential of d is by
// (2.5 |d| + 2) 2^-24 of itself (the argument, its product with log2(e), that
// constant; exp2).  A softmax adds its sum, off by the terms' own errors (their
// mean |d| is at most log(1024)) and up to 37 additions in a row, and the quotient: by
// less than 64 2^-24 of the row's largest probability, 1 / z, in all (|d| e^-|d| <
// 0.4).  A sigmoid is off by less than 2^-21.  The sums with the bias round once more.
// The sums of two groups that 64 bits do not tell apart either come as they are
// rounded there.
//
// What that costs goes by the values, since the bounds are those of the row's
// largest (kernel us, 65536 tokens): a bias of 0 and 8 of 256 normal logits of
// standard deviation 1, 3, 5, 8 take 36, 39, 57 and 104 with softmax, 28, 30, 38
// and 146 with sigmoid (scores near 1 differ by less than 2^-21); with biases of
// 0.05 33-37 and 28-29.  A large finite value in a row (-1e9 for what is masked)
// takes all steps of the scale where the low value is the row's smallest: with
// groups, or no more lanes than slots (8 of 64 experts 9 -> 108, 2 of 8 3.6 ->
// 58, 8 of 256 19 as without); -inf costs nothing.
//
// A token's result depends on its row and on E, top_k and the groups alone,
// not on the batch it comes in.
//
// Bound by its vector instructions: 65536 tokens, 8 of 256 experts, fp32 19-20 us
// (15 for the bytes), 546 instructions a wave of four tokens, 300 of them in the
// selection; bf16 17.2; with sigmoid scores, a bias and groups 35 (1003).  16
// lanes of 16 logits take fewer of them a token than 64 of 4 (the lane steps are
// shared by four tokens).
// ---------------------------------------------------------------------------
template <int V>
SFP8_DEV float max_nan(const float (&x)[V]) {
  float m = x[0];
#pragma unroll
  for (int j = 1; j + 1 < V; j += 2) m = max3_nan(m, x[j], x[j + 1]);
  return V % 2 ? m : __builtin_elementwise_maximum(m, x[V - 1]);
}

// sigmoid(x) without its sum's cancellation: e^x / (1 + e^x) below 0.
SFP8_DEV float sigmoid_of(float x) {
  const float en = exp_fast(-fabsf(x));
  return (x > 0.0f ? 1.0f : en) * __builtin_amdgcn_rcpf(1.0f + en);
}

template <int L, int V, bool BIAS>
__global__ __launch_bounds__(256, 4) void moe_route_kernel(const RouteArgs a, int log_g, int gs, int idx_bits) {
  extern __shared__ __align__(16) uint64_t lds[];
  constexpr int kTok = 64 / L;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tl = lane & (L - 1), tok = lane / L;  // lane of the token, token of the wave
  const int G = 1 << log_g;
  const RouteLayout lay{G, gs, tl >> log_g, tl & (G - 1)};
  const bool in_group = lay.g < a.groups;
  const float ninf = -__builtin_inff();
  const bool half16 = !BIAS && a.dtype != kF32;  // ranks hold the whole logit
  const bool softmax = a.score == kSoftmax;
  const bool two_best = a.groups > 1 && a.group_best == 2;
  const bool scores = BIAS || !a.renorm || two_best;  // scores of all experts, not of the chosen alone
  const int first = lay.g * lay.gs;                   // the group's first expert
  const int64_t t0 = ((int64_t)blockIdx.x * 4 + wave) * kTok;
  if (t0 >= a.T) return;
  const bool on = t0 + tok < a.T && !(a.mask && !a.mask[t0 + tok]);
  const int64_t row = t0 * a.ld + tok * a.ld;
  float l[V];
  load_logits<V>(l, a.logits, a.dtype, row + first, lay, on && in_group);
  float mine_max = max_nan<V>(l);             // NaN if one is
  bool odd = !(mine_max < __builtin_inff());  // selected again in 64 bits
  float m = ninf, z = 1.0f;
  if (softmax && scores) {
    m = lanes_max<L>(mine_max);
    z = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) z += l[j] == ninf ? 0.0f : exp_fast(l[j] - m);
    z = lanes_sum<L>(z);
  }
  // the order values
  float o[V];
  float err = 0.0f;  // how far a score may be off
  if constexpr (BIAS) {
    const float rz = __builtin_amdgcn_rcpf(z);
    err = softmax ? 0x1p-18f * rz : 0x1p-21f;
    float bias[V];
    load_logits<V>(bias, a.bias, kF32, first, lay, in_group);
#pragma unroll
    for (int c = 0; c < V / 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 4 * c + i;
        const float sc = softmax ? exp_fast(l[j] - m) * rz : sigmoid_of(l[j]);
        o[j] = l[j] == ninf ? ninf : sc + bias[j];
      }
    mine_max = max_nan<V>(o);
    odd |= !(mine_max < __builtin_inff());
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = l[j];
  }
  bool kept = in_group;
  if (a.groups > 1) {
    // the best two of this lane, then of its group
    float b1 = ninf, b2 = ninf;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      b2 = __builtin_amdgcn_fmed3f(b1, b2, o[j]);
      b1 = fmaxf(b1, o[j]);
    }
    const auto merge = [&](float p1, float q1, float p2, float q2) {
      b1 = fmaxf(p1, q1);
      b2 = fmaxf(fminf(p1, q1), fmaxf(p2, q2));
    };
    float p1, q1, p2, q2;
    if constexpr (L > 1)
      if (G > 1) share_f<1>(b1, p1, q1), share_f<1>(b2, p2, q2), merge(p1, q1, p2, q2);
    if constexpr (L > 2)
      if (G > 2) share_f<2>(b1, p1, q1), share_f<2>(b2, p2, q2), merge(p1, q1, p2, q2);
    if constexpr (L > 4)
      if (G > 4) share_f<4>(b1, p1, q1), share_f<4>(b2, p2, q2), merge(p1, q1, p2, q2);
    if constexpr (L > 8)
      if (G > 8) share_f<8>(b1, p1, q1), share_f<8>(b2, p2, q2), merge(p1, q1, p2, q2);
    if constexpr (L > 16)
      if (G > 16) share_f<16>(b1, p1, q1), share_f<16>(b2, p2, q2), merge(p1, q1, p2, q2);
    if constexpr (L > 32)
      if (G > 32) share_f<32>(b1, p1, q1), share_f<32>(b2, p2, q2), merge(p1, q1, p2, q2);
    float val = b1, tol = 0.0f;  // tol: how far two groups' values may be off together
    if constexpr (BIAS) {
      const float big = lanes_max<L>(b1 == ninf ? 0.0f : fmaxf(fabsf(b1), b2 == ninf ? 0.0f : fabsf(b2)));
      tol = (two_best ? 4.0f : 2.0f) * (err + 0x1p-23f * big);
    }
    if (two_best && b1 != ninf) {
      if constexpr (!BIAS) {
        b1 = softmax ? exp_fast(b1 - m) : sigmoid_of(b1);  // z is the same for all
        b2 = b2 == ninf ? ninf : softmax ? exp_fast(b2 - m) : sigmoid_of(b2);
      }
      val = b1 + (b2 == ninf ? 0.0f : b2);
      // of scores: (2.5 |d| + 8) 2^-24 of each, |d| < 104 (below, they vanish)
      if constexpr (!BIAS) tol = 0x1p-14f * val + 0x1p-120f;
    }
    int rank = 0, over = 0, near = 0;
    for (int j = 1; j < L >> log_g; ++j) {
      const int from = (tl + j * G) & (L - 1);
      const float other = __shfl(val, (lane & ~(L - 1)) + from, 64);
      rank += other > val || (other == val && from < tl);
      over += other > val + tol;
      near += other >= val - tol;
    }
    kept = in_group && val != ninf && rank < a.top_groups;
    const bool unsure = on && tol > 0.0f && val != ninf && over < a.top_groups && near >= a.top_groups;
    if (BIAS && softmax) {
      odd |= unsure;
    } else if (__any(unsure)) {
      // a group at the border of those kept: the groups' values in 64 bits
      double d1 = ninf, d2 = ninf;
#pragma unroll 1
      for (int j = 0; j < V; ++j) {
        const int mem = lay.member(j >> 2) + (j & 3);
        if (!(on && in_group && mem < gs)) continue;
        const float x = load_as_f32(a.logits, a.dtype, row + first + mem);
        if (x == ninf) continue;
        const double ex = exp(softmax ? (double)x - (double)m : -(double)x);
        const double v = softmax ? ex : 1.0 / (1.0 + ex) + (BIAS ? (double)a.bias[first + mem] : 0.0);
        d2 = fmax(d2, fmin(d1, v));
        d1 = fmax(d1, v);
      }
      for (int s = 1; s < G; s <<= 1) {
        const double o1 = __shfl_xor(d1, s, 64), o2 = __shfl_xor(d2, s, 64);
        d2 = fmax(fmin(d1, o1), fmax(d2, o2));
        d1 = fmax(d1, o1);
      }
      const double v = two_best && d2 != ninf ? d1 + d2 : d1;
      int place = 0;
      for (int j = 1; j < L >> log_g; ++j) {
        const int from = (tl + j * G) & (L - 1);
        const double other = __shfl(v, (lane & ~(L - 1)) + from, 64);
        place += other > v || (other == v && from < tl);
      }
      kept = in_group && v != ninf && place < a.top_groups;
    }
  }
  // the keys: rank << idx_bits, and the inverted index (a padding lane's index may
  // be past the mask: its key wraps to one that comes after all others)
  const uint32_t idx_mask = (1u << idx_bits) - 1, idx_top = idx_mask - (uint32_t)first;
  uint32_t key[V], least;  // keys from `least` on can be taken
  float gap = 0.0f;        // ranks that are no further apart may be in the wrong order
  if (half16) {
    const bool bf16 = a.dtype == kBf16;
    least = (bf16 ? 0x80u : 0x400u) << idx_bits;  // above -inf
    const uint32_t keep = kept ? ~idx_mask : 0u;
    const int down = 16 - idx_bits;
#pragma unroll
    for (int c = 0; c < V / 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = l[4 * c + i] + 0.0f;  // -0 is 0
        const uint32_t b = bf16 ? __float_as_uint(x) : f32_to_half_bits(x) << 16;
        const uint32_t ord = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
        key[4 * c + i] = (ord >> down & keep) | (idx_top - (uint32_t)(lay.member(c) + i));
      }
  } else {
    least = 1u << idx_bits;
    const float hi = lanes_max<L>(mine_max);
    float lo = ninf;
    if (a.groups == 1 && L > a.k) {
      lo = lanes_min<L>(mine_max);
      // What is below it by no more than two values' errors has a rank too, so
      // that it is found among the near neighbours (3: and the steps to here).
      if constexpr (BIAS) lo -= 3.0f * (err + 0x1p-23f * fmaxf(fabsf(lo), fabsf(hi)));
    }
    if (__any(lo == ninf)) {  // a lane without an expert, a group that is out: the row's smallest
      float least_o = __builtin_inff();
#pragma unroll
      for (int j = 0; j < V; ++j) least_o = fminf(least_o, o[j] == ninf ? least_o : o[j]);
      least_o = lanes_min<L>(least_o);
      lo = lo == ninf ? least_o : lo;  // each token its own
    }
    const float range = hi - lo;
    // below 2^(31 - idx_bits) at the largest value, by two steps and the quotient's 2^-22
    const float steps = (float)(1u << (31 - idx_bits)) * (1.0f - 0x1p-19f) - 4.0f;
    // A range outside 2^+-100 is left to 64 bits, and its keys are all alike: a scale
    // that overflows would take a rank past 31 bits, among the keys that wrap.
    const bool fits = range > 0x1p-100f && range < 0x1p100f;
    odd |= range > 0.0f && !fits;
    const float scale = kept && fits ? steps * __builtin_amdgcn_rcpf(range) : 0.0f;
    const float base = kept ? 0x1p23f + 1.0f : 0x1p23f;
    // a value's error, and three steps for the scale's own roundings
    if constexpr (BIAS) gap = 2.0f * (err + 0x1p-23f * fmaxf(fabsf(lo), fabsf(hi))) * lanes_max<L>(scale) + 3.0f;
#pragma unroll
    for (int c = 0; c < V / 4; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = fmaxf(__builtin_fmaf(o[4 * c + i] - lo, scale, base), 0x1p23f);
        key[4 * c + i] = __float_as_uint(x) << idx_bits | (idx_top - (uint32_t)(lay.member(c) + i));
      }
  }
  // the first top_k keys, lane s of the token keeping that of slot s, and the one after them
  uint32_t top = 1u << 31, mine = 0u, after = 0u;
  const int rounds = a.k + (half16 ? 0 : 1);
  for (int s = 0; s < rounds; ++s) {
    uint32_t r = 0u;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint32_t x = key[j] - top;
      r = x > r ? x : r;
    }
    r = reduce_max_u<L>(r);
    top += r;
    if (s < a.k) mine = s == tl ? top : mine;  // uniform
    else after = top;
  }
  int e = mine >= least ? (int)(idx_mask - (mine & idx_mask)) : -1;
  float le = e >= 0 ? load_as_f32(a.logits, a.dtype, row + e) : ninf;
  if (!half16) {
    const uint32_t up = __shfl_up(mine, 1, 64);
    const uint32_t last = __shfl(mine, (lane & ~(L - 1)) + a.k - 1, 64);
    const auto close = [&](uint32_t x, uint32_t y) {  // x comes first
      return y >= least && (float)((x >> idx_bits) - (y >> idx_bits)) <= gap;
    };
    if (__any((tl > 0 && tl < a.k && close(up, mine)) || close(last, after))) {
      // Near neighbours with the same logit and bias are equal, and in the order
      // of their indices: that leaves those that differ, among the chosen or
      // between the last of them and the rest.
      const float be = BIAS && e >= 0 ? a.bias[e] : 0.0f;
      const float la = __shfl_up(le, 1, 64), ba = __shfl_up(be, 1, 64);
      bool differ = tl > 0 && e >= 0 && close(up, mine) && !(la == le && ba == be);
      const int from = (lane & ~(L - 1)) + a.k - 1;
      const float ll = __shfl(le, from, 64), bl = __shfl(be, from, 64);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (key[j] < last && close(last, key[j])) {
          const int x = (int)(idx_mask - (key[j] & idx_mask));
          differ |= load_as_f32(a.logits, a.dtype, row + x) != ll || (BIAS && a.bias[x] != bl);
        }
      differ = lanes_max<L>(differ && on ? 1.0f : 0.0f) > 0.0f;  // the token
      if (__any(differ)) {
        // The chosen and the next few, each in a lane, by their values in 64 bits.
        // What is not among them is further from the last chosen than the errors.
        const int n = a.k + 4 < L ? a.k + 4 : L;
        uint32_t cand = tl == a.k ? after : mine, tail = after;
        for (int s = a.k + 1; s < n; ++s) {
          uint32_t r = 0u;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const uint32_t x = key[j] - tail;
            r = x > r ? x : r;
          }
          tail += reduce_max_u<L>(r);
          cand = s == tl ? tail : cand;
        }
        // tail > last: the keys are used up
        odd |= differ && ((tail < last && close(last, tail)) || (BIAS && softmax));
        const bool is = tl < n && cand >= least && (tl < a.k || cand < last);
        const int ce = is ? (int)(idx_mask - (cand & idx_mask)) : -1;
        double val = 0.0;
        if (is) {
          val = load_as_f32(a.logits, a.dtype, row + ce);
          if constexpr (BIAS) val = 1.0 / (1.0 + exp(-val)) + (double)a.bias[ce];
        }
        int place = 0;
        for (int j = 0; j < n; ++j) {
          const int src = (lane & ~(L - 1)) + j;
          const double ov = __shfl(val, src, 64);
          const int oe = __shfl(ce, src, 64);
          place += oe >= 0 && (ov > val || (ov == val && oe < ce));
        }
        // those that are none stay in the lanes behind
        const int to = (lane & ~(L - 1)) + (is ? place : tl);
        const int placed = __builtin_amdgcn_ds_permute(to << 2, ce);
        if (differ) {
          e = tl < a.k ? placed : -1;
          le = e >= 0 ? load_as_f32(a.logits, a.dtype, row + e) : ninf;
        }
      }
    }
  }
  const uint64_t any_odd = __ballot(odd && on);
  if (any_odd) {  // wave uniform
    for (int i = 0; i < kTok; ++i) {
      if (!(any_odd >> (i * L) & (L == 64 ? ~0ull : (1ull << L) - 1))) continue;
      const int again = __shfl(route_exact(a, t0 + i, lds + wave * ((3 * a.E + 1) / 2)), tl, 64);
      if (tok == i) {
        e = tl < a.k ? again : -1;
        le = e >= 0 ? load_as_f32(a.logits, a.dtype, row + e) : ninf;
      }
    }
  }
  // the weights
  const bool live = e >= 0;
  float w;
  if (softmax) {
    const float top_l = a.renorm ? lanes_max<L>(le) : m;
    w = live ? exp_fast(le - top_l) : 0.0f;
    w *= __builtin_amdgcn_rcpf(a.renorm ? lanes_sum<L>(w) : z);
  } else {
    const float en = exp_fast(-fabsf(le)), low = fminf(le, 0.0f);
    const float top_l = a.renorm ? lanes_max<L>(low) : 0.0f;
    w = live ? exp_fast(low - top_l) * __builtin_amdgcn_rcpf(1.0f + en) : 0.0f;
    if (a.renorm) w *= __builtin_amdgcn_rcpf(lanes_sum<L>(w));
  }
  if (t0 + tok < a.T && tl < a.k) {
    const int64_t base = t0 * a.k;
    const int at = tok * a.k + tl;
    (a.weights + base)[at] = live ? a.scale * w : 0.0f;
    (a.selected + base)[at] = e;
    if (a.picked) (a.picked + base)[at] = live ? le : 0.0f;
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

// The gradient of the logits, L lanes a token and V values a lane as the
// forward has them without groups.  Lane s of a token computes what slot s gives
// its expert, from the chosen logits alone; the plain softmax also reads the
// row again, for p of every expert.  The row is put together in LDS (zeros or
// the dense part, then the slots' values) and written whole, once: bound by
// those bytes (65536 x 256 fp32 13.5 us, 5.0 TB/s, the plain softmax 22.6, 5.9 read
// and written; 65536 x 8 bf16 3.4).
template <int L, int V>
__global__ __launch_bounds__(256) void moe_route_bwd_kernel(const RouteBwdArgs a) {
  __shared__ __align__(16) float rows[256 * V];
  constexpr int kTok = 64 / L;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tl = lane & (L - 1);
  const int64_t t0 = ((int64_t)blockIdx.x * 4 + wave) * kTok;
  if (t0 >= a.T) return;
  const int64_t t = t0 + lane / L;
  const bool on = t < a.T;
  const float ninf = -__builtin_inff();
  const RouteLayout lay{L, a.E, 0, tl};
  float* row = rows + (wave * kTok + lane / L) * (L * V);
  const int64_t sel = on && tl < a.k ? a.selected[t * a.k + tl] : -1;
  const bool live = sel >= 0 && sel < a.E;
  const float g = live ? a.scale * a.dweights[t * a.k + tl] : 0.0f;
  const float le = live ? a.picked[t * a.k + tl] : ninf;
  const bool dense = a.score == kSoftmax && !a.renorm;
  float mine, d[V];
#pragma unroll
  for (int j = 0; j < V; ++j) d[j] = 0.0f;
  if (dense) {
    float l[V], m = ninf, z = 0.0f;
    load_logits<V>(l, a.logits, a.dtype, t * a.ld, lay, on);
#pragma unroll
    for (int j = 0; j < V; ++j) m = fmaxf(m, l[j]);
    m = lanes_max<L>(m);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      l[j] = l[j] == ninf ? 0.0f : exp_fast(l[j] - m);
      z += l[j];
    }
    z = lanes_sum<L>(z);
    const float some = lanes_max<L>(live ? 1.0f : 0.0f);
    const float p = live ? exp_fast(le - m) / z : 0.0f;
    mine = g * p;
    const float dot = lanes_sum<L>(mine), f = -dot / z;
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = some > 0.0f ? f * l[j] : 0.0f;
  } else {
    const float en = exp_fast(-fabsf(le)), r = 1.0f / (1.0f + en);
    if (a.renorm) {
      const float x = a.score == kSoftmax ? le : fminf(le, 0.0f);
      const float top = lanes_max<L>(x);
      float q = live ? exp_fast(x - top) : 0.0f;
      if (a.score == kSigmoid) q *= r;
      const float w = q / lanes_sum<L>(q);
      const float share = live ? w : 0.0f;
      mine = share * (g - lanes_sum<L>(g * share));
      if (a.score == kSigmoid) mine *= (le > 0.0f ? en : 1.0f) * r;  // 1 - sigmoid
    } else {
      mine = g * en * r * r;
    }
  }
#pragma unroll
  for (int c = 0; c < V / 4; ++c)
    *reinterpret_cast<floatx4*>(row + lay.member(c)) = floatx4{d[4 * c], d[4 * c + 1], d[4 * c + 2], d[4 * c + 3]};
  __builtin_amdgcn_wave_barrier();
  if (live) row[sel] += mine;  // each expert at most once in a token
  __builtin_amdgcn_wave_barrier();
  if (!on) return;
#pragma unroll
  for (int c = 0; c < V / 4; ++c) {
    const int mem = lay.member(c);
    if (mem >= a.E) continue;
    const floatx4 v = *reinterpret_cast<const floatx4*>(row + mem);
    const int64_t at = t * a.E + mem;
    if (mem + 4 <= a.E && a.dtype == kF32) {
      *reinterpret_cast<floatx4_any*>(reinterpret_cast<float*>(a.dlogits) + at) = v;
    } else if (mem + 4 <= a.E) {
      const intx2 o = a.dtype == kBf16 ? intx2{(int)pack2_bf16(v[0], v[1]), (int)pack2_bf16(v[2], v[3])}
                                       : intx2{(int)(f32_to_half_bits(v[0]) | f32_to_half_bits(v[1]) << 16),
                                               (int)(f32_to_half_bits(v[2]) | f32_to_half_bits(v[3]) << 16)};
      *reinterpret_cast<intx2_any*>(reinterpret_cast<uint16_t*>(a.dlogits) + at) = o;
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (mem + i < a.E) store_f32_as(a.dlogits, a.dtype, at + i, v[i]);
    }
  }
}

// ---------------------------------------------------------------------------
// Expert order: a stable counting sort of the R = T * k slots by expert, bin E
// holding the slots that name none.  A work-group takes `chunk` consecutive
// slots, wave w of it the w-th sixteenth.  One launch counts each group's bins;
// in the second every group adds up the counts itself (at most 256 rows of E +
// 1, from the L2), which is cheaper than a third launch that would scan them.
// Up to 4096 slots are one group and one launch.  Bound by its launches and by
// the chain of steps of the second (counts, sums, places), 24 bytes a slot are a
// sixth of the time: 524288 slots of 256 experts 15.2 us, 131072 of 8 9.2, 64 of
// 128 4.2.
// ---------------------------------------------------------------------------
constexpr int kOrderWaves = 16;
constexpr int kOrderThreads = 64 * kOrderWaves;
constexpr int kOrderBlocks = 256;

// Slots per work-group: a multiple of its threads, at most kOrderBlocks groups.
// Below that many, shorter groups are faster where the counts that each adds up
// stay short too (us at 2048 and 4096 slots a group: 131072 slots of 8 experts
// 9.3 and 11.0, of 256 experts 11.4 and 13.1; 524288 slots of 1024 experts 29
// and 23), and one group alone up to 4096 (7.8, against 8.7 in two).
inline int64_t order_chunk(int64_t R, int64_t E) {
  const int64_t c = (R + kOrderBlocks - 1) / kOrderBlocks;
  const int64_t few = R <= 4096 || E >= 512 ? 4096 : 2048;
  const int64_t least = c < few ? few : c;
  return (least + kOrderThreads - 1) / kOrderThreads * kOrderThreads;
}
// Parts of the rows that are added up side by side: 3 (257 columns) to 32.
__host__ __device__ inline int order_parts(int cols) { return kOrderThreads / cols < 32 ? kOrderThreads / cols : 32; }
// Bins of a row of counts: E + 1, in whole 16-byte units.
__host__ __device__ inline int order_stride(int E) { return (E + 4) / 4 * 4; }

SFP8_DEV int order_bin(const int64_t* sel, int64_t i, int E) {
  const int64_t e = sel[i];
  return e >= 0 && e < E ? (int)e : E;
}

// counts[b][e]: slots of work-group b that name expert e.
__global__ __launch_bounds__(kOrderThreads) void moe_order_count_kernel(const int64_t* __restrict__ sel, int64_t R,
                                                                         int64_t chunk, int E,
                                                                         int* __restrict__ counts) {
  extern __shared__ __align__(16) int hist[];
  const int stride = order_stride(E);
  for (int e = threadIdx.x; e < stride; e += kOrderThreads) hist[e] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * chunk;
  const int64_t i1 = i0 + chunk < R ? i0 + chunk : R;
#pragma unroll 4
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kOrderThreads) atomicAdd(&hist[order_bin(sel, i, E)], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < stride; e += kOrderThreads) counts[(int64_t)blockIdx.x * stride + e] = hist[e];
}

__global__ __launch_bounds__(kOrderThreads) void moe_order_place_kernel(
    const int64_t* __restrict__ sel, int64_t R, int64_t chunk, int k, int E, const int* __restrict__ counts,
    int64_t* __restrict__ token_index, int64_t* __restrict__ inverse, int* __restrict__ offsets) {
  // next[wave][bin]: the next row of each bin, per wave; then, while the counts
  // are added up, the sums of each part of the work-group
  extern __shared__ __align__(16) int next[];
  __shared__ int part[kOrderWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nb = gridDim.x, bins = E + 1;
  const int stride = order_stride(E), cols = stride / 4;
  const int parts = counts ? order_parts(cols) : 0;
  int* sums = next + kOrderWaves * stride;              // [parts][2][stride]: all rows, the rows before this group's
  for (int e = threadIdx.x; e < kOrderWaves * stride; e += kOrderThreads) next[e] = 0;
  if (counts && (int)threadIdx.x < parts * cols) {
    const int p = threadIdx.x / cols, c = threadIdx.x % cols;
    intx4 before = {0, 0, 0, 0}, after = {0, 0, 0, 0};
    const intx4* row = reinterpret_cast<const intx4*>(counts) + p * cols + c;
    const int step = parts * cols, own = blockIdx.x;
    int b = p;
#pragma unroll 8
    for (; b < own; b += parts, row += step) before += *row;
#pragma unroll 8
    for (; b < nb; b += parts, row += step) after += *row;
    *reinterpret_cast<intx4*>(sums + (2 * p) * stride + 4 * c) = before + after;
    *reinterpret_cast<intx4*>(sums + (2 * p + 1) * stride + 4 * c) = before;
  }
  __syncthreads();
  int* mine = next + wave * stride;
  const int64_t per = chunk / kOrderWaves;
  const int64_t i0 = (int64_t)blockIdx.x * chunk + wave * per;
  const int64_t i1 = i0 + per < R ? i0 + per : R;
#pragma unroll 4
  for (int64_t i = i0 + lane; i < i1; i += 64) atomicAdd(&mine[order_bin(sel, i, E)], 1);
  __syncthreads();
  // start of each bin: the totals of the bins before it, then this bin's slots of earlier work-groups
  for (int e0 = 0, carry = 0; e0 < bins; e0 += kOrderThreads) {
    const int e = e0 + threadIdx.x;
    int total = 0, before = 0;
    if (e < bins) {
      if (counts) {
        for (int p = 0; p < parts; ++p) {
          total += sums[(2 * p) * stride + e];
          before += sums[(2 * p + 1) * stride + e];
        }
      } else {
#pragma unroll
        for (int w = 0; w < kOrderWaves; ++w) total += next[w * stride + e];
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
#pragma unroll
    for (int w = 0; w < kOrderWaves; ++w) {
      base += w < wave ? part[w] : 0;
      all += part[w];
    }
    __syncthreads();
    carry = all;
    if (e < bins) {
      if (blockIdx.x == 0 && e < E) offsets[e] = base + scan;
      int at = base + scan - total + before;
#pragma unroll
      for (int w = 0; w < kOrderWaves; ++w) {
        const int c = next[w * stride + e];
        next[w * stride + e] = at;
        at += c;
      }
    }
  }
  __syncthreads();
  int bits = 0;
  while ((1 << bits) < bins) ++bits;
  for (int i = (int)i0 + lane; i - lane < (int)i1; i += 64) {  // R <= 2^30
    const bool in = i < (int)i1;
    const int e = in ? order_bin(sel, i, E) : 0;
    uint64_t same = __ballot(in);  // the lanes of this step with the same bin
    for (int b = 0; b < bits; ++b) {
      const int bit = __builtin_amdgcn_sbfe(e, b, 1);  // 0 or -1
      const uint64_t y = __ballot(bit);
      same &= ~(y ^ (uint64_t)(int64_t)bit);
    }
    const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
    const int row = in ? mine[e] + rank : 0;
    __builtin_amdgcn_wave_barrier();
    if (in && rank == 0) mine[e] = row + __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (in) {
      inverse[i] = e < E ? row : -1;
      token_index[row] = (uint32_t)i / (uint32_t)k;
    }
  }
}

// ---------------------------------------------------------------------------
// Combine: out[t] = sum over j of w[t, j] rows[inv[t, j]], summed in 32 bits in
// slot order and rounded once; slots whose row is out of range add nothing.
// `lanes` lanes (a power of two) take one token, U elements at a time.
// ---------------------------------------------------------------------------
// How a row is cut into units: one element each (rows shorter than 16 bytes),
// whole aligned 16-byte units, or 16 bytes at any address, where the last unit
// of a row ends with it and so may hold elements of the one before.
enum : int { kSingle = 0, kWhole = 1, kAny = 2 };

template <int DT, int CUT>
struct Unit {  // U consecutive elements as fp32
  static constexpr int U = CUT == kSingle ? 1 : DT == kF32 ? 4 : 8;
  float x[U];
  // First element of the unit that would start at d; the elements before d - first are another unit's too.
  SFP8_DEV static int64_t first(int64_t d, int64_t D) { return CUT == kAny && d > D - U ? D - U : d; }
  // as they are in memory: what a load in flight holds
  struct Raw {
    intx4 v;
    SFP8_DEV void load(const void* p, int64_t i) {
      if constexpr (CUT == kSingle) {
        v[0] = DT == kF32 ? reinterpret_cast<const int*>(p)[i] : reinterpret_cast<const uint16_t*>(p)[i];
      } else {
        const char* at = reinterpret_cast<const char*>(p) + i * (DT == kF32 ? 4 : 2);
        if constexpr (CUT == kWhole) v = *reinterpret_cast<const intx4*>(at);
        else v = *reinterpret_cast<const intx4_any*>(at);
      }
    }
    // the same of data that is read once
    SFP8_DEV void load_once(const void* p, int64_t i) {
      const char* at = reinterpret_cast<const char*>(p) + i * (DT == kF32 ? 4 : 2);
      if constexpr (CUT == kSingle) load(p, i);
      else if constexpr (CUT == kWhole) v = __builtin_nontemporal_load(reinterpret_cast<const intx4*>(at));
      else v = __builtin_nontemporal_load(reinterpret_cast<const intx4_any*>(at));
    }
  };
  SFP8_DEV Unit() = default;
  SFP8_DEV explicit Unit(const Raw& r) {
    if constexpr (DT == kF32) {
#pragma unroll
      for (int q = 0; q < U; ++q) x[q] = __uint_as_float((uint32_t)r.v[q]);
    } else {
#pragma unroll
      for (int q = 0; q < U; ++q) {
        const uint32_t b = ((uint32_t)r.v[q >> 1] >> (16 * (q & 1))) & 0xffffu;
        x[q] = DT == kBf16 ? bf16_bits_to_f32(b) : half_bits_to_f32(b);
      }
    }
  }
  // ONCE: past the caches
  template <bool ONCE = false>
  SFP8_DEV void store(void* p, int64_t i) const {
    if constexpr (CUT == kSingle) {
      store_f32_as(p, DT, i, x[0]);
    } else {
      intx4 o;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if constexpr (DT == kF32) o[q] = (int)__float_as_uint(x[q]);
        else if constexpr (DT == kBf16) o[q] = (int)pack2_bf16(x[2 * q], x[2 * q + 1]);
        else o[q] = (int)(f32_to_half_bits(x[2 * q]) | f32_to_half_bits(x[2 * q + 1]) << 16);
      }
      char* at = reinterpret_cast<char*>(p) + i * (DT == kF32 ? 4 : 2);
      if constexpr (CUT == kAny && ONCE) __builtin_nontemporal_store(o, reinterpret_cast<intx4_any*>(at));
      else if constexpr (CUT == kAny) *reinterpret_cast<intx4_any*>(at) = o;
      else if constexpr (ONCE) __builtin_nontemporal_store(o, reinterpret_cast<intx4*>(at));
      else *reinterpret_cast<intx4*>(at) = o;
    }
  }
};

// One unit a lane: `lanes` (a power of two) lanes for the D / U units of a token
// where those are fewer than a wave's, else whole waves.  K slots' rows are in
// flight at once.  Bound by the rows' bytes (65536 tokens of 2 rows of 1024 67
// us, 6.0 TB/s; of 1022, at odd addresses, 70); for few tokens by two dependent
// loads, which one unit a lane keeps from repeating (8 tokens of 8 of 2048 3.2).
template <int DT, int CUT, int K, bool NT>
__global__ __launch_bounds__(256) void moe_combine_kernel(const void* __restrict__ rows, int64_t R, int64_t D,
                                                          const float* __restrict__ weights,
                                                          const int64_t* __restrict__ inv, int64_t T, int k,
                                                          void* __restrict__ out, int lanes, int waves) {
  using X = Unit<DT, CUT>;
  int64_t t, d0, step;
  if (lanes == 64) {  // `waves` waves a token
    const uint32_t w = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const uint32_t tt = w / (uint32_t)waves;
    t = tt;
    d0 = ((int64_t)(w - tt * (uint32_t)waves) * 64 + (threadIdx.x & 63)) * X::U;
    step = (int64_t)waves * 64 * X::U;
  } else {
    t = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    d0 = (int64_t)(threadIdx.x & (lanes - 1)) * X::U;
    step = (int64_t)lanes * X::U;
  }
  if (t >= T) return;
  for (int64_t at = d0; at < D; at += step) {  // once, but for launches beyond 2^32 work-items
    const int64_t d = X::first(at, D);
    X acc;
#pragma unroll
    for (int q = 0; q < X::U; ++q) acc.x[q] = 0.0f;
    for (int j0 = 0; j0 < k; j0 += K) {
      int64_t r[K];
      float w[K];
      typename X::Raw v[K];
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const bool in = j0 + j < k;
        r[j] = in ? inv[t * k + j0 + j] : -1;
        w[j] = in ? weights[t * k + j0 + j] : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < K; ++j) {
        if (r[j] >= 0 && r[j] < R) {
          NT ? v[j].load_once(rows, r[j] * D + d) : v[j].load(rows, r[j] * D + d);
        } else {
          w[j] = 0.0f;
          v[j].v = intx4{0, 0, 0, 0};
        }
      }
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const X x(v[j]);
#pragma unroll
        for (int q = 0; q < X::U; ++q) acc.x[q] = __builtin_fmaf(w[j], x.x[q], acc.x[q]);
      }
    }
    acc.store(out, t * D + d);
  }
}

// ---------------------------------------------------------------------------
// Which slots name a row, from the slots alone: the combine's backward pass must
// write every row once, whatever the slots name.  of_row[r] becomes a slot that
// names row r, and many[s] says of that slot whether there are others.  Neither
// is cleared first, since what is left in of_row[r] proves itself: a number s
// there is right if slot s names row r.  The slot that wrote last took the one
// before it out of of_row[r], if there was one; a stale number can only pass for
// another slot of the row where it is one.  Which of a row's slots comes last
// changes from run to run, the gradients do not: one slot is the row's own, and
// of several any one adds up all of them, in order.  4 bytes a slot, scattered,
// and 9 in a row: 131072 slots 5 us.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void moe_row_slots_kernel(const int64_t* __restrict__ inv, int64_t slots, int64_t R,
                                                            uint32_t* __restrict__ of_row, uint8_t* __restrict__ many) {
  const int64_t s = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (s >= slots) return;
  const int64_t r = inv[s];
  if (r < 0 || r >= R) return;
  const uint32_t before = atomicExch(of_row + r, (uint32_t)s);
  many[s] = before < slots && before != (uint32_t)s && inv[before] == r;
}

// drows[r] = the sum over the slots of row r, in order, of w dout: a whole wave.
template <int DT>
SFP8_DEV void sum_slots(const void* dout, int64_t D, const float* weights, const int64_t* inv, int64_t slots, int k,
                        int64_t r, void* drows) {
  const int lane = threadIdx.x & 63;
  for (int64_t d0 = lane; d0 - lane < D; d0 += 256) {
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t b = 0; b < slots; b += 64) {
      uint64_t found = __ballot(b + lane < slots && inv[b + lane] == r);
      for (; found; found &= found - 1) {
        const int64_t s = b + __builtin_ctzll(found);
        const float w = weights[s];
        const int64_t at = (int64_t)((uint32_t)s / (uint32_t)k) * D;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (d0 + 64 * q < D) acc[q] = __builtin_fmaf(w, load_as_f32(dout, DT, at + d0 + 64 * q), acc[q]);
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (d0 + 64 * q < D) store_f32_as(drows, DT, r * D + d0 + 64 * q, acc[q]);
  }
}

// drows[inv[t, j]] = w[t, j] dout[t], dw[t, j] = <dout[t], rows[inv[t, j]]>
// (either may be null).  With of_row and many (moe_row_slots_kernel) a row that
// several slots name gets the sum of theirs and one that none names zeros;
// without them each row below offsets[E - 1] is one slot's, and those from there
// on get zeros.  One wave a slot, or `lanes` lanes (a power of two) where a row
// has fewer units: the lanes of a token's slots share its gradient through the
// caches.  Bound by the rows' bytes, read and written (65536 tokens of 2 rows of
// 1024 103 us, 6.5 TB/s; 131072 of 2 of 128 32, in whole waves 53).
template <int DT, int CUT, bool NT, bool WIDE>
__global__ __launch_bounds__(256) void moe_combine_bwd_kernel(
    const void* __restrict__ dout, const void* __restrict__ rows, int64_t R, int64_t D,
    const float* __restrict__ weights, const int64_t* __restrict__ inv, int64_t slots, int k,
    const int* __restrict__ offsets, int E, const uint32_t* __restrict__ of_row, const uint8_t* __restrict__ many,
    void* __restrict__ drows, float* __restrict__ dweights, int lanes) {
  using X = Unit<DT, CUT>;
  const int per = WIDE ? 1 : 64 / lanes;  // slots of a wave
  const int sub = WIDE ? threadIdx.x & 63 : threadIdx.x & (lanes - 1);
  const int64_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int64_t first = wave * per + (WIDE ? 0 : (threadIdx.x & 63) / lanes), step = (int64_t)gridDim.x * 4 * per;
  const int64_t stride = (int64_t)(WIDE ? 64 : lanes) * X::U;
  for (int64_t s = first; s - first < slots - wave * per; s += step) {  // the lanes of a wave together
    const bool in = s < slots;
    const int64_t t = (uint32_t)s / (uint32_t)k, r = in ? inv[s] : -1;
    float dot = 0.0f;
    bool sum = false;
    if (r >= 0 && r < R) {
      const float w = weights[s];
      // the slot that writes the row, and whether it alone names it
      const uint32_t owner = of_row ? of_row[r] : (uint32_t)s, others = of_row ? many[s] : 0u;
#pragma unroll 2
      for (int64_t at = (int64_t)sub * X::U; at < D; at += stride) {
        const int64_t d = X::first(at, D);
        typename X::Raw rg, rv;
        rg.load(dout, t * D + d);
        if (dweights) NT ? rv.load_once(rows, r * D + d) : rv.load(rows, r * D + d);
        X g(rg);
        if (dweights) {
          const X v(rv);
#pragma unroll
          for (int q = 0; q < X::U; ++q)
            dot = CUT != kAny || q >= at - d ? __builtin_fmaf(g.x[q], v.x[q], dot) : dot;
        }
        uint32_t writes = owner == (uint32_t)s && !others && drows;
        asm volatile("" : "+v"(writes));  // asked for here, with the rows' loads in flight (before them: 4 us of 100 more)
        if (writes) {
#pragma unroll
          for (int q = 0; q < X::U; ++q) g.x[q] *= w;
          g.template store<NT>(drows, r * D + d);
        }
      }
      sum = owner == (uint32_t)s && others;
    }
    if (dweights) {
      if constexpr (WIDE) dot = lanes_sum<64>(dot);
      else
        for (int o = 1; o < lanes; o <<= 1) dot += __shfl_xor(dot, o, 64);
      if (in && sub == 0) dweights[s] = dot;
    }
    for (uint64_t left = __ballot(sum && sub == 0); left; left &= left - 1)  // seldom any
      sum_slots<DT>(dout, D, weights, inv, slots, k, __shfl(r, __builtin_ctzll(left), 64), drows);
  }
  if (!drows) return;
  X zero;
#pragma unroll
  for (int q = 0; q < X::U; ++q) zero.x[q] = 0.0f;
  if (of_row) {
    const int lane = threadIdx.x & 63;
    for (int64_t b = wave * 64; b < R; b += (int64_t)gridDim.x * 256) {  // 64 rows a wave
      bool none = false;
      if (b + lane < R) {
        const uint32_t s = of_row[b + lane];
        none = !(s < slots && inv[s] == b + lane);
      }
      for (uint64_t left = __ballot(none); left; left &= left - 1) {
        const int64_t r = b + __builtin_ctzll(left);
        for (int64_t d = (int64_t)lane * X::U; d < D; d += 64 * X::U) zero.store(drows, r * D + X::first(d, D));
      }
    }
    return;
  }
  int64_t used = offsets[E - 1];
  used = used < 0 ? 0 : used;
  for (int64_t r = used + first; r < R; r += step)
    for (int64_t d = (int64_t)sub * X::U; d < D; d += stride) zero.store(drows, r * D + X::first(d, D));
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

// Calls F<dtype, cut>.
template <template <int, int> class F, int DT, typename... A>
void by_cut(int cut, A... args) {
  cut == kWhole ? F<DT, kWhole>::run(args...) : cut == kAny ? F<DT, kAny>::run(args...) : F<DT, kSingle>::run(args...);
}
template <template <int, int> class F, typename... A>
void by_type(int dtype, int cut, A... args) {
  if (dtype == kF32) by_cut<F, kF32>(cut, args...);
  else if (dtype == kBf16) by_cut<F, kBf16>(cut, args...);
  else by_cut<F, kF16>(cut, args...);
}
int row_cut(int dtype, int64_t D, bool aligned) {
  const int64_t unit = dtype == kF32 ? 4 : 8;
  return D < unit ? kSingle : D % unit == 0 && aligned ? kWhole : kAny;
}

// Lanes of a token and of a group, and values of a lane: the fewest lanes that
// hold every group at 16 values each and have one for every slot; at most 64,
// with up to 32 values where the number of groups is no power of two.
struct RouteShape {
  int L, G, V;
};
RouteShape route_shape(int64_t E, int64_t groups, int64_t k) {
  int gp = 1;
  while (gp < groups) gp *= 2;
  const int gs = (int)(E / groups);
  int G = 1;
  while ((G * 16 < gs || gp * G < k) && gp * G < 64) G *= 2;
  const int need = (gs + G - 1) / G;  // above 16 where gp lanes of G would be more than a wave
  return {gp * G, G, need <= 4 ? 4 : need <= 8 ? 8 : need <= 16 ? 16 : 32};
}

template <int L, int V>
void route_run(const RouteArgs& a, const RouteShape& sh, hipStream_t st) {
  int idx_bits = 8;  // at least: a rank's mantissa then leaves its exponent behind (moe_route_kernel)
  while ((1 << idx_bits) < a.E) ++idx_bits;
  const int64_t per = 4 * (64 / L);  // tokens of a work-group
  const dim3 grid((unsigned)((a.T + per - 1) / per));
  const size_t lds = 4 * (size_t)((3 * a.E + 1) / 2) * 8;  // of each wave: an order value and a logit per expert
  const int gs = a.E / a.groups;
  int log_g = 0;
  while ((1 << log_g) < sh.G) ++log_g;
  if (a.bias) hipLaunchKernelGGL((moe_route_kernel<L, V, true>), grid, dim3(256), lds, st, a, log_g, gs, idx_bits);
  else hipLaunchKernelGGL((moe_route_kernel<L, V, false>), grid, dim3(256), lds, st, a, log_g, gs, idx_bits);
}
template <int L, int V>
void route_run(const RouteBwdArgs& a, const RouteShape&, hipStream_t st) {
  const int64_t per = 4 * (64 / L);
  hipLaunchKernelGGL((moe_route_bwd_kernel<L, V>), dim3((unsigned)((a.T + per - 1) / per)), dim3(256), 0, st, a);
}
template <int L, class Args>
void route_run_l(const Args& a, const RouteShape& sh, hipStream_t st) {
  if (sh.V == 4) route_run<L, 4>(a, sh, st);
  else if (sh.V == 8) route_run<L, 8>(a, sh, st);
  else route_run<L, 16>(a, sh, st);
}
template <class Args>
void route_by_shape(const Args& a, const RouteShape& sh, hipStream_t st) {
  switch (sh.L) {
    case 1: return route_run_l<1>(a, sh, st);
    case 2: return route_run_l<2>(a, sh, st);
    case 4: return route_run_l<4>(a, sh, st);
    case 8: return route_run_l<8>(a, sh, st);
    case 16: return route_run_l<16>(a, sh, st);
    case 32: return route_run_l<32>(a, sh, st);
    default: return route_run_l<64>(a, sh, st);
  }
}
void route_launch(const RouteArgs& a, hipStream_t st) {
  const RouteShape sh = route_shape(a.E, a.groups, a.k);
  if (sh.V == 32) return route_run<64, 32>(a, sh, st);
  route_by_shape(a, sh, st);
}
void route_bwd_launch(const RouteBwdArgs& a, hipStream_t st) { route_by_shape(a, route_shape(a.E, 1, a.k), st); }

// What no longer fits the last-level cache passes it by: the rows, and in the
// backward pass their gradients too.  us with that and without, by MiB of rows
// and results, forward: 192 36.5 and 31.7, 216 40.6 and 34.2, 288 52 and 52, 336
// 59 and 64, 384 66.5 and 77, 768 124 and 146; backward: 160 31 and 27, 240 42 and
// 39, 272 53 and 55, 320 51 and 61, 480 80 and 98, 640 102 and 129, 1088 211 and 225.
constexpr int64_t kLastLevelCache = (int64_t)256 << 20;

template <int DT, int CUT>
struct Combine {
  template <int K>
  static void go(const void* rows, int64_t R, int64_t D, const float* w, const int64_t* inv, int64_t T, int k, void* out,
                 hipStream_t st) {
    constexpr int U = Unit<DT, CUT>::U;
    const int64_t units = (D + U - 1) / U, most = ((int64_t)1 << 25) / T;  // waves: 2^31 work-items
    const int64_t waves = (units + 63) / 64 < most ? (units + 63) / 64 : most;
    int lanes = 64;
    while (lanes > 1 && lanes / 2 >= units) lanes /= 2;
    const int64_t per = 256 / lanes, blocks = lanes == 64 ? (T * waves + 3) / 4 : (T + per - 1) / per;
    const auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, st, rows, R, D, w, inv, T, k, out, lanes,
                         (int)waves);
    };
    constexpr bool kPast = CUT != kSingle;
    if (kPast && (R + T) * D * (DT == kF32 ? 4 : 2) > kLastLevelCache) launch(moe_combine_kernel<DT, CUT, K, kPast>);
    else launch(moe_combine_kernel<DT, CUT, K, false>);
  }
  static void run(const void* rows, int64_t R, int64_t D, const float* w, const int64_t* inv, int64_t T, int k,
                  void* out, hipStream_t st) {
    if (k == 1) go<1>(rows, R, D, w, inv, T, k, out, st);
    else if (k == 2) go<2>(rows, R, D, w, inv, T, k, out, st);
    else if (k <= 4) go<4>(rows, R, D, w, inv, T, k, out, st);
    else go<8>(rows, R, D, w, inv, T, k, out, st);
  }
};

template <int DT, int CUT>
struct CombineBwd {
  static void run(const void* dout, const void* rows, int64_t R, int64_t D, const float* w, const int64_t* inv,
                  int64_t T, int k, const int* offsets, int E, const uint32_t* of_row, const uint8_t* many,
                  void* drows, float* dw, hipStream_t st) {
    constexpr int U = Unit<DT, CUT>::U;
    int lanes = 64;
    while (lanes > 1 && (int64_t)(lanes / 2) * U >= D) lanes /= 2;
    const int64_t slots = T * k, work = slots > 0 ? slots : R, most = (int64_t)1 << 22;
    const int64_t per = 4 * (64 / lanes), need = (work + per - 1) / per, nb = need < most ? need : most;
    const auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)nb), dim3(256), 0, st, dout, rows, R, D, w, inv, slots, k, offsets, E,
                         of_row, many, drows, dw, lanes);
    };
    constexpr bool kPast = CUT != kSingle;
    const bool past = kPast && (2 * R + T) * D * (DT == kF32 ? 4 : 2) > kLastLevelCache;
    if (lanes == 64) {
      if (past) launch(moe_combine_bwd_kernel<DT, CUT, kPast, true>);
      else launch(moe_combine_bwd_kernel<DT, CUT, false, true>);
    } else {
      if (past) launch(moe_combine_bwd_kernel<DT, CUT, kPast, false>);
      else launch(moe_combine_bwd_kernel<DT, CUT, false, false>);
    }
  }
};

int combine_bwd_check(const void* dout, const void* rows, int dtype, int64_t R, int64_t D, const float* weights,
                      const int64_t* inverse, int64_t T, int64_t top_k, const float* dweights) {
  if ((T > 0 && (!dout || !weights || !inverse)) || (R > 0 && dweights && T > 0 && !rows)) return kErrNullPointer;
  if (R < 0 || T < 0 || T > kMaxTokens || D <= 0 || top_k <= 0 || top_k > kRouteMaxK || bad_dtype(dtype))
    return kErrBadShape;
  return kOk;
}
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
  route_launch(a, (hipStream_t)stream);
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
  route_bwd_launch(a, (hipStream_t)stream);
  return route_status();
}

int64_t sfp8_moe_expert_order_workspace_ints(int64_t R, int64_t E) {
  if (R < 0 || R > (int64_t)1 << 30 || E <= 0 || E > kRouteMaxExperts) return -1;
  const int64_t chunk = order_chunk(R, E), nb = (R + chunk - 1) / chunk;
  return nb > 1 ? nb * order_stride((int)E) : 0;
}

int sfp8_moe_expert_order(const int64_t* selected, int64_t R, int64_t top_k, int64_t E, int64_t* token_index,
                          int64_t* inverse, int* offsets, int* ws, int64_t ws_ints, void* stream) {
  if (!offsets || (R > 0 && (!selected || !token_index || !inverse))) return kErrNullPointer;
  const int64_t need = sfp8_moe_expert_order_workspace_ints(R, E);
  if (need < 0 || top_k <= 0 || R % top_k) return kErrBadShape;
  if (need > 0 && (!ws || ws_ints < need)) return kErrWorkspaceTooSmall;
  const int64_t chunk = order_chunk(R, E);
  const int64_t nb = R > chunk ? (R + chunk - 1) / chunk : 1;
  const int stride = order_stride((int)E);
  // 16 rows of bins, and up to 1024 columns of 16 bytes for two sums
  const size_t lds = (size_t)kOrderWaves * stride * 4 + (nb > 1 ? (size_t)order_parts(stride / 4) * 2 * stride * 4 : 0);
  if (const int rc = route_allow_lds(moe_order_place_kernel, lds)) return rc;
  if (nb > 1)
    hipLaunchKernelGGL(moe_order_count_kernel, dim3((unsigned)nb), dim3(kOrderThreads), (size_t)stride * 4,
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
  const int cut = row_cut(dtype, D, al16(rows) && al16(out));
  by_type<Combine>(dtype, cut, rows, R, D, weights, inverse, T, (int)top_k, out, (hipStream_t)stream);
  return route_status();
}

int sfp8_moe_combine_bwd(const void* dout, const void* rows, int dtype, int64_t R, int64_t D, const float* weights,
                         const int64_t* inverse, int64_t T, int64_t top_k, const int* offsets, int64_t E, void* drows,
                         float* dweights, void* stream) {
  if (const int rc = combine_bwd_check(dout, rows, dtype, R, D, weights, inverse, T, top_k, dweights)) return rc;
  if (drows && !offsets) return kErrNullPointer;
  if (E <= 0) return kErrBadShape;
  if ((T == 0 && R == 0) || (!drows && !dweights)) return kOk;
  const int cut = row_cut(dtype, D, al16(rows) && al16(dout) && al16(drows));
  by_type<CombineBwd>(dtype, cut, dout, rows, R, D, weights, inverse, T, (int)top_k, offsets, (int)E,
                      (const uint32_t*)nullptr, (const uint8_t*)nullptr, drows, dweights, (hipStream_t)stream);
  return route_status();
}

// of_row of every row, then a byte of many for every slot
int64_t sfp8_moe_combine_bwd_any_workspace_ints(int64_t R, int64_t T, int64_t top_k) {
  if (R < 0 || T < 0 || T > kMaxTokens || top_k <= 0 || top_k > kRouteMaxK) return -1;
  return R + (T * top_k + 3) / 4;
}

int sfp8_moe_combine_bwd_any(const void* dout, const void* rows, int dtype, int64_t R, int64_t D, const float* weights,
                             const int64_t* inverse, int64_t T, int64_t top_k, void* drows, float* dweights, int* ws,
                             int64_t ws_ints, void* stream) {
  if (const int rc = combine_bwd_check(dout, rows, dtype, R, D, weights, inverse, T, top_k, dweights)) return rc;
  if ((T == 0 && R == 0) || (!drows && !dweights)) return kOk;
  uint32_t* of_row = nullptr;
  uint8_t* many = nullptr;
  if (drows && R > 0) {
    if (!ws || ws_ints < sfp8_moe_combine_bwd_any_workspace_ints(R, T, top_k)) return kErrWorkspaceTooSmall;
    of_row = (uint32_t*)ws;
    many = (uint8_t*)(ws + R);
    const int64_t slots = T * top_k;
    if (slots > 0)
      hipLaunchKernelGGL(moe_row_slots_kernel, dim3((unsigned)((slots + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                         inverse, slots, R, of_row, many);
  } else if (!dweights) {
    return kOk;  // no rows
  }
  const int cut = row_cut(dtype, D, al16(rows) && al16(dout) && al16(drows));
  by_type<CombineBwd>(dtype, cut, dout, rows, R, D, weights, inverse, T, (int)top_k, (const int*)nullptr, 0,
                      (const uint32_t*)of_row, (const uint8_t*)many, R > 0 ? drows : nullptr, dweights,
                      (hipStream_t)stream);
  return route_status();
}

}  // extern "C"
