// A mixture-of-experts layer for a few tokens (gfx950): router, selection,
// gate and up with SwiGLU, down, weighted sum.
//
//   l = x R^T (64-bit sums); the top_k experts and weights as moe_route has
//   them, ordered by values in 64 bits
//   h_j = silu(x Wg_j^T) * (x Wu_j^T);  out = sum_j w_j h_j Wd_j^T
//
// With at most 64 tokens the layer is bound by the bytes of the experts that
// are taken, so each of their weights is read once for all tokens and goes from
// memory to registers (16 bytes a lane); the products run on the bf16 matrix
// cores with the weights as first operand and up to 16 tokens as second.
// Weights are bf16, or MXFP4 codes (mx4.h) that become bf16 values in
// registers, which hold them exactly; x stays bf16 in both.
// Four launches: logits; one work-group that selects and sorts the slots by
// expert; gate and up; down and the sum.
#include <type_traits>

#include "mx4.h"

namespace sfp8 {

constexpr int kMaxTokens = 64, kMaxExperts = 1024, kMaxTopK = 64;
constexpr int kSlots = kMaxTokens * kMaxTopK;

struct DecodeArgs {
  const uint16_t* x;
  int64_t ldx;
  int T, E, k, D, I;
  const void* router;
  int router_f32;
  const uint8_t *gu, *gu_scales, *down, *down_scales;  // scales NULL: bf16 rows
  const float* bias;
  const uint8_t* mask;
  int score, groups, top_groups, group_best, renorm;
  float scale;
  int64_t* selected;
  uint16_t* out;
  // workspace
  double* low;      // [T, E]
  float* weights;   // [T, k]
  int* plan;        // number of experts taken; their index, first slot; the slots by expert
  uint16_t* h;      // [T * k][2][I]: h and what its rounding to bf16 left
};

// plan: [0] experts taken; [1 + a] expert; [1 + n + a] begin (one past the last too); then the slots
__host__ __device__ inline int plan_most(int T, int E, int k) { return T * k < E ? T * k : E; }
struct Plan {
  const int* p;
  int most;
  SFP8_DEV int count() const { return p[0]; }
  SFP8_DEV int expert(int a) const { return p[1 + a]; }
  SFP8_DEV int begin(int a) const { return p[1 + most + a]; }
  SFP8_DEV const int* slots() const { return p + 2 + 2 * most; }
};

SFP8_DEV double wave_sum(double v) { return wave_sum_f64(v); }
SFP8_DEV double wave_max_or_nan(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const double w = __shfl_xor(v, o, 64);
    v = (w > v || w != w) ? w : v;
  }
  return v;
}

// ---------------------------------------------------------------------------
// Logits: a work-group takes one expert and up to 8 tokens, its four waves a
// quarter of the width each.  Sums in 64 bits, so that the order of two experts
// is that of the exact sums but for 2^-50 of their size.
// ---------------------------------------------------------------------------
constexpr int kLogitTokens = 8;

__global__ __launch_bounds__(256) void decode_logits_kernel(DecodeArgs a) {
  __shared__ double part[4][kLogitTokens];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int e = blockIdx.x, t0 = blockIdx.y * kLogitTokens, n = min(kLogitTokens, a.T - t0);
  double acc[kLogitTokens];
#pragma unroll
  for (int t = 0; t < kLogitTokens; ++t) acc[t] = 0.0;
  for (int d = 8 * threadIdx.x; d < a.D; d += 8 * 256) {
    double w[8];
    if (a.router_f32) {
      const float* p = reinterpret_cast<const float*>(a.router) + (int64_t)e * a.D + d;
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = (double)p[j];
    } else {
      const Eight<kMxBf16> v = load8<kMxBf16>(a.router, (int64_t)e * a.D + d);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = (double)__uint_as_float(j & 1 ? v.w[j / 2] & 0xffff0000u : v.w[j / 2] << 16);
    }
#pragma unroll
    for (int t = 0; t < kLogitTokens; ++t) {
      if (t < n) {
        const Eight<kMxBf16> v = load8<kMxBf16>(a.x, (t0 + t) * a.ldx + d);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          acc[t] = fma((double)__uint_as_float(j & 1 ? v.w[j / 2] & 0xffff0000u : v.w[j / 2] << 16), w[j], acc[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < kLogitTokens; ++t) {
    if (t < n) {
      const double s = wave_sum(acc[t]);
      if (lane == 0) part[wave][t] = s;
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < n)
    a.low[(int64_t)(t0 + threadIdx.x) * a.E + e] =
        (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
}

// ---------------------------------------------------------------------------
// Selection
// ---------------------------------------------------------------------------
// Order values as unsigned keys: NaN above all, -0 as 0; 0 stands for an expert
// that cannot be taken (-inf, or taken already).
SFP8_DEV uint64_t order_key(double v) {
  if (v != v) return ~0ull;
  if (v == -__builtin_inf()) return 0;
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

template <int CTRL>
SFP8_DEV uint32_t dpp_max(uint32_t x) {
  const uint32_t y = (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xf, 0xf, true);
  return x > y ? x : y;
}
// the maximum over the wave, in every lane
SFP8_DEV uint32_t wave_max_u(uint32_t x) {
  x = dpp_max<0xB1>(x);
  x = dpp_max<0x4E>(x);
  x = dpp_max<0x141>(x);
  x = dpp_max<0x140>(x);
  const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = p[0] > p[1] ? p[0] : p[1];
  const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return q[0] > q[1] ? q[0] : q[1];
}

struct Scores {  // of one token
  const double* low;
  int score;
  double top, sum;  // softmax: the largest logit (NaN if there is one), the sum of exp(l - top)
  SFP8_DEV double operator()(int e) const {
    return score == 0 ? exp(low[e] - top) / sum : 1.0 / (1.0 + exp(-low[e]));
  }
};

// One wave selects for one token; keys: E of LDS.  chosen[j] = expert or -1, w[j] its weight (lane j).
SFP8_DEV void select_token(const DecodeArgs& a, int t, uint64_t* keys, int& chosen, float& weight) {
  const int lane = threadIdx.x & 63;
  const double* low = a.low + (int64_t)t * a.E;
  chosen = -1;
  weight = 0.f;
  if (a.mask && !a.mask[t]) return;
  Scores s{low, a.score, 0.0, 1.0};
  const bool all_scores = a.bias || (a.groups > 1 && a.group_best == 2) || !a.renorm;
  if (a.score == 0 && all_scores) {
    double m = -__builtin_inf(), z = 0.0;
    for (int e = lane; e < a.E; e += 64) m = (low[e] > m || low[e] != low[e]) ? low[e] : m;
    s.top = wave_max_or_nan(m);
    for (int e = lane; e < a.E; e += 64) z += exp(low[e] - s.top);
    s.sum = wave_sum(z);
  }
  for (int e = lane; e < a.E; e += 64) {
    const double l = low[e];
    keys[e] = l == -__builtin_inf() ? 0 : order_key(a.bias ? s(e) + (double)a.bias[e] : l);
  }
  __builtin_amdgcn_wave_barrier();
  __threadfence_block();
  if (a.groups > 1) {
    const int size = a.E / a.groups;
    uint64_t mine = 0;
    if (lane < a.groups) {
      uint64_t k1 = 0, k2 = 0;
      int e1 = -1, e2 = -1;
      for (int e = lane * size; e < (lane + 1) * size; ++e) {
        const uint64_t key = keys[e];
        if (key > k1) k2 = k1, e2 = e1, k1 = key, e1 = e;
        else if (key > k2) k2 = key, e2 = e;
      }
      mine = k1;
      if (a.group_best == 2 && e1 >= 0) {
        double v = s(e1) + (a.bias ? (double)a.bias[e1] : 0.0);
        if (e2 >= 0) v += s(e2) + (a.bias ? (double)a.bias[e2] : 0.0);
        mine = order_key(v);
      }
    }
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint64_t other = __shfl(mine, g, 64);
      rank += other > mine || (other == mine && g < lane);
    }
    const uint64_t kept = __ballot(lane < a.groups && mine != 0 && rank < a.top_groups);
    for (int e = lane; e < a.E; e += 64)
      if (!(kept >> (e / size) & 1)) keys[e] = 0;
    __builtin_amdgcn_wave_barrier();
    __threadfence_block();
  }
  // lane's own best among e = lane, lane + 64, ..: the lowest of equals
  uint64_t best = 0;
  int at = 0;
  const auto rescan = [&]() {
    best = 0, at = lane;
    for (int e = lane; e < a.E; e += 64)
      if (keys[e] > best) best = keys[e], at = e;
  };
  rescan();
  for (int j = 0; j < a.k; ++j) {
    const uint32_t hi = wave_max_u((uint32_t)(best >> 32));
    bool in = (uint32_t)(best >> 32) == hi;
    uint64_t who = __ballot(in);
    if (who & (who - 1)) {
      const uint32_t lo = wave_max_u(in ? (uint32_t)best : 0u);
      in = in && (uint32_t)best == lo;
      who = __ballot(in);
      if (who & (who - 1)) {
        const uint32_t first = ~wave_max_u(in ? ~(uint32_t)at : 0u);
        who = __ballot(in && (uint32_t)at == first);
      }
    }
    const int win = __builtin_ctzll(who);
    const uint32_t top_hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(best >> 32), win);
    const uint32_t top_lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)best, win);
    if ((top_hi | top_lo) == 0) break;  // nobody is left
    const int e = __builtin_amdgcn_readlane(at, win);
    if (lane == j) chosen = e;
    if (lane == win) {
      keys[e] = 0;
      rescan();
    }
  }
  // weights: shares of the chosen, in 64 bits
  const bool there = chosen >= 0;
  const double l = there ? low[chosen] : 0.0;
  double share;
  if (!a.renorm) {
    share = there ? s(chosen) : 0.0;
  } else {
    // sigmoid(l) = exp(min(l, 0)) / (1 + exp(-|l|)): over exp of the largest min(l, 0) it cannot vanish for all
    const double low_part = a.score == 0 ? l : (l > 0.0 ? 0.0 : l);
    const double m = wave_max_or_nan(there ? low_part : -__builtin_inf());
    const double v = exp(low_part - m);
    const double part = there ? (a.score == 0 ? v : v / (1.0 + exp(-fabs(l)))) : 0.0;
    share = part / wave_sum(part);
  }
  weight = there ? (float)((double)a.scale * share) : 0.f;
}

// One work-group: a wave a token, then a thread an expert for the plan.
__global__ __launch_bounds__(1024) void decode_select_kernel(DecodeArgs a) {
  extern __shared__ __align__(16) uint64_t keys[];  // [waves][E]
  __shared__ short sel[kSlots];
  __shared__ int wave_slots[16], wave_experts[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  for (int t = wave; t < a.T; t += waves) {
    int chosen;
    float w;
    select_token(a, t, keys + (int64_t)wave * a.E, chosen, w);
    if (lane < a.k) {
      sel[t * a.k + lane] = (short)chosen;
      a.selected[t * a.k + lane] = chosen;
      a.weights[t * a.k + lane] = w;
    }
  }
  __syncthreads();
  // experts in blocks of the work-group's threads; slots and experts before each
  const int slots = a.T * a.k, most = plan_most(a.T, a.E, a.k);
  int* out = a.plan + 2 + 2 * most;
  int base_slots = 0, base_experts = 0;
  for (int e0 = 0; e0 < a.E; e0 += blockDim.x) {
    const int e = e0 + tid;
    int n = 0;
    for (int s = 0; s < slots; ++s) n += sel[s] == e;
    int before = n, live = n > 0;  // inclusive sums over the lanes
    int upto = live;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int p = __shfl_up(before, o, 64), q = __shfl_up(upto, o, 64);
      if (lane >= o) before += p, upto += q;
    }
    if (lane == 63) wave_slots[wave] = before, wave_experts[wave] = upto;
    __syncthreads();
    int first = base_slots, rank = base_experts, all_slots = 0, all_experts = 0;
    for (int w = 0; w < waves; ++w) {
      if (w < wave) first += wave_slots[w], rank += wave_experts[w];
      all_slots += wave_slots[w], all_experts += wave_experts[w];
    }
    first += before - n, rank += upto - live;
    if (live) {
      a.plan[1 + rank] = e;
      a.plan[1 + most + rank] = first;
      for (int s = 0, i = first; s < slots; ++s)
        if (sel[s] == e) out[i++] = s;
    }
    base_slots += all_slots, base_experts += all_experts;
    __syncthreads();
  }
  if (tid == 0) {
    a.plan[0] = base_experts;
    a.plan[1 + most + base_experts] = base_slots;
  }
}

// ---------------------------------------------------------------------------
// The experts
// ---------------------------------------------------------------------------
SFP8_DEV bf16x8 as_bf16x8(const Eight<kMxBf16>& v) {
  return __builtin_bit_cast(bf16x8, intx4{(int)v.w[0], (int)v.w[1], (int)v.w[2], (int)v.w[3]});
}
SFP8_DEV bf16x8 load_bf16x8(const uint16_t* p) { return as_bf16x8(load8<kMxBf16>(p, 0)); }
SFP8_DEV bf16x8 zero_unless(bool ok, bf16x8 v) {
  const intx4 i = __builtin_bit_cast(intx4, v);
  return __builtin_bit_cast(bf16x8, intx4{ok ? i[0] : 0, ok ? i[1] : 0, ok ? i[2] : 0, ok ? i[3] : 0});
}
SFP8_DEV floatx4 mfma16(bf16x8 w, bf16x8 x, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(w, x, c, 0, 0, 0);
}

// How a lane (row r of 16, quarter q) reads a stretch of K of its weight row:
// kStep values a wave and step, kPieces pieces of 8 a lane, piece j at value
// at(q, j) of the stretch.
template <bool W4>
struct Stretch {
  static constexpr int kStep = W4 ? 128 : 64, kPieces = W4 ? 4 : 2;
  static SFP8_DEV int at(int q, int j) { return kPieces * 8 * q + 8 * j; }
  bf16x8 w[kPieces];
};

// Rows of one expert's matrix.
template <bool W4>
struct WeightRows;
template <>
struct WeightRows<false> {
  const uint16_t* p;  // [rows, K]
  int64_t K;
  SFP8_DEV WeightRows(const uint8_t* base, const uint8_t*, int64_t e, int64_t rows, int64_t k)
      : p(reinterpret_cast<const uint16_t*>(base) + e * rows * k), K(k) {}
  // step s of row n; past K (a multiple of 8) the last piece again, whose product the caller zeroes
  template <bool TAIL>
  SFP8_DEV void read(int64_t n, int s, int q, Stretch<false>& f) const {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      int64_t k = (int64_t)s * 64 + Stretch<false>::at(q, j);
      bool ok = true;
      if (TAIL) ok = k < K, k = ok ? k : K - 8;
      f.w[j] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const intx4*>(p + n * K + k));
      if (TAIL) f.w[j] = zero_unless(ok, f.w[j]);
    }
  }
};
template <>
struct WeightRows<true> {
  const uint8_t *codes, *scales;  // [slabs][rows rounded up][64], [..][4]
  int64_t rows;
  SFP8_DEV WeightRows(const uint8_t* c, const uint8_t* s, int64_t e, int64_t r, int64_t k) : rows(mx_rows(r)) {
    codes = c + e * mx_slabs(k) * rows * 64;
    scales = s + e * mx_slabs(k) * rows * 4;
  }
  template <bool TAIL>
  SFP8_DEV void read(int64_t n, int s, int q, Stretch<true>& f) const {
    const intx4 c = *reinterpret_cast<const intx4*>(codes + (s * rows + n) * 64 + 16 * q);
    const uint32_t e = *reinterpret_cast<const uint32_t*>(scales + (s * rows + n) * 4) >> (8 * q) & 255u;
    const float v = mx_scale_value(e);
#pragma unroll
    for (int j = 0; j < 4; ++j) f.w[j] = bf16_of_codes8((uint32_t)c[j], v);
  }
};

// A token's (or slot's) values beside them.
template <bool W4, bool TAIL>
SFP8_DEV void read_values(const uint16_t* row, int K, int s, int q, Stretch<W4>& f) {
#pragma unroll
  for (int j = 0; j < Stretch<W4>::kPieces; ++j) {
    int k = s * Stretch<W4>::kStep + Stretch<W4>::at(q, j);
    bool ok = true;
    if (TAIL) ok = k < K, k = ok ? k : K - 8;
    f.w[j] = load_bf16x8(row + k);
    if (TAIL) f.w[j] = zero_unless(ok, f.w[j]);
  }
}

// Gate and up of 16 columns of h for all slots of one expert: eight waves share
// the width, their sums meet in LDS in the order of the waves.  NB: blocks of
// 16 slots that an expert can have.
template <bool W4, int NB>
__global__ __launch_bounds__(512) void decode_gateup_kernel(DecodeArgs a) {
  constexpr int W = 8;
  __shared__ __align__(16) float red[W][2][NB * 16][20];
  const Plan plan{a.plan, plan_most(a.T, a.E, a.k)};
  const int which = blockIdx.y;
  if (which >= plan.count()) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, q = lane >> 4;
  const int e = plan.expert(which), begin = plan.begin(which), n = plan.begin(which + 1) - begin;
  const int* slots = plan.slots() + begin;
  const int i0 = 16 * blockIdx.x, D = a.D, I = a.I;
  const WeightRows<W4> w(a.gu, a.gu_scales, e, 2 * (int64_t)I, D);
  const int64_t grow = min(i0 + r, I - 1), urow = I + grow;
  const uint16_t* xrow[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int s = 16 * b + r;  // a lane without a slot goes along with the first
    xrow[b] = a.x + (slots[s < n ? s : 0] / a.k) * a.ldx;
  }
  floatx4 g[NB], u[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) g[b] = u[b] = floatx4{0.f, 0.f, 0.f, 0.f};
  const auto step = [&](auto tail, int s) {
    constexpr bool TAIL = decltype(tail)::value;
    Stretch<W4> fg, fu, fx;
    w.template read<TAIL>(grow, s, q, fg);
    w.template read<TAIL>(urow, s, q, fu);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (b == 0 || 16 * b < n) {
        read_values<W4, TAIL>(xrow[b], D, s, q, fx);
#pragma unroll
        for (int j = 0; j < Stretch<W4>::kPieces; ++j) {
          g[b] = mfma16(fg.w[j], fx.w[j], g[b]);
          u[b] = mfma16(fu.w[j], fx.w[j], u[b]);
        }
      }
    }
  };
  const int full = D / Stretch<W4>::kStep;
  for (int s = wave; s < full; s += W) step(std::false_type{}, s);
  if (D % Stretch<W4>::kStep && wave == full % W) step(std::true_type{}, full);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    *reinterpret_cast<floatx4*>(&red[wave][0][16 * b + r][4 * q]) = g[b];
    *reinterpret_cast<floatx4*>(&red[wave][1][16 * b + r][4 * q]) = u[b];
  }
  __syncthreads();
  for (int i = tid; i < n * 16; i += 64 * W) {
    const int s = i >> 4, c = i & 15;
    float gs = 0.f, us = 0.f;
#pragma unroll
    for (int v = 0; v < W; ++v) gs += red[v][0][s][c], us += red[v][1][s][c];
    if (i0 + c < I) {
      const float h = gs * sigmoid_fast(gs) * us, hi = round_bf16(h);
      uint16_t* p = a.h + (int64_t)slots[s] * 2 * I + i0 + c;
      p[0] = (uint16_t)f32_to_bf16_bits(h);
      // an infinity or a NaN leaves nothing to be added
      p[I] = (uint16_t)f32_to_bf16_bits(__builtin_isfinite(hi) ? h - hi : 0.f);
    }
  }
}

// Down and the weighted sum for 16 columns of the output: the steps of all
// experts that are taken, in their order, are dealt out to the waves in even
// runs.  A wave adds each expert's sums times the slots' weights to its own
// totals of all tokens (LDS), and the waves' totals meet in their order: every
// weight is read once, and no sum depends on the order of arrival.
template <bool W4, int NB>
__global__ __launch_bounds__(512) void decode_down_kernel(DecodeArgs a) {
  constexpr int W = 8;
  extern __shared__ __align__(16) float totals[];  // [W][T][16]
  const Plan plan{a.plan, plan_most(a.T, a.E, a.k)};
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, q = lane >> 4;
  const int n0 = 16 * blockIdx.x, D = a.D, I = a.I, T = a.T;
  float* mine = totals + wave * T * 16;
  for (int i = lane; i < T * 4; i += 64) reinterpret_cast<floatx4*>(mine)[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  const int steps = (I + Stretch<W4>::kStep - 1) / Stretch<W4>::kStep;
  const int64_t all = (int64_t)plan.count() * steps;
  const int lo = (int)(all * wave / W), hi = (int)(all * (wave + 1) / W);
  const int64_t row = min(n0 + r, D - 1);
  for (int at = lo; at < hi;) {
    const int which = at / steps, s0 = at - which * steps, s1 = min(steps, s0 + hi - at);
    at += s1 - s0;
    const int e = plan.expert(which), begin = plan.begin(which), n = plan.begin(which + 1) - begin;
    const int* slots = plan.slots() + begin;
    const WeightRows<W4> w(a.down, a.down_scales, e, D, I);
    const uint16_t* hrow[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int s = 16 * b + r;
      hrow[b] = a.h + (int64_t)slots[s < n ? s : 0] * 2 * I;
    }
    floatx4 acc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = floatx4{0.f, 0.f, 0.f, 0.f};
    const auto step = [&](auto tail, int s) {
      constexpr bool TAIL = decltype(tail)::value;
      Stretch<W4> fw, f0, f1;
      w.template read<TAIL>(row, s, q, fw);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        if (b == 0 || 16 * b < n) {
          read_values<W4, TAIL>(hrow[b], I, s, q, f0);
          read_values<W4, TAIL>(hrow[b] + I, I, s, q, f1);
#pragma unroll
          for (int j = 0; j < Stretch<W4>::kPieces; ++j) {
            acc[b] = mfma16(fw.w[j], f0.w[j], acc[b]);
            acc[b] = mfma16(fw.w[j], f1.w[j], acc[b]);
          }
        }
      }
    };
    const int full = I / Stretch<W4>::kStep;
    for (int s = s0; s < min(s1, full); ++s) step(std::false_type{}, s);
    if (s1 > full) step(std::true_type{}, full);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int s = 16 * b + r;
      if (s < n) {
        const int slot = slots[s];
        const float wt = a.weights[slot];
        floatx4* p = reinterpret_cast<floatx4*>(mine + (slot / a.k) * 16 + 4 * q);
        floatx4 t = *p;
#pragma unroll
        for (int v = 0; v < 4; ++v) t[v] = __builtin_fmaf(wt, acc[b][v], t[v]);
        *p = t;
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < T * 8; i += 64 * W) {
    const int t = i >> 3, c = 2 * (i & 7);
    float v0 = 0.f, v1 = 0.f;
#pragma unroll
    for (int v = 0; v < W; ++v) v0 += totals[(v * T + t) * 16 + c], v1 += totals[(v * T + t) * 16 + c + 1];
    if (n0 + c < D) *reinterpret_cast<uint32_t*>(a.out + (int64_t)t * D + n0 + c) = pack2_bf16(v0, v1);
  }
}

inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

struct DecodeSpace {
  int64_t low, weights, plan, h, all;
  DecodeSpace(int64_t T, int64_t E, int64_t k, int64_t I) {
    low = 0;
    weights = low + up256(T * E * 8);
    plan = weights + up256(T * k * 4);
    h = plan + up256((2 + 2 * plan_most((int)T, (int)E, (int)k) + T * k) * 4);
    all = h + T * k * 2 * I * 2;
  }
};

inline bool decode_sizes_ok(int64_t T, int64_t E, int64_t k, int64_t D, int64_t I) {
  return T >= 0 && T <= kMaxTokens && E >= 1 && E <= kMaxExperts && k >= 1 && k <= kMaxTopK && k <= E && D >= 8 &&
         D % 8 == 0 && D <= 1 << 20 && I >= 8 && I % 8 == 0 && I <= 1 << 20;
}

template <bool W4, int NB>
int launch_experts(const DecodeArgs& a, hipStream_t s) {
  decode_gateup_kernel<W4, NB><<<dim3((a.I + 15) / 16, plan_most(a.T, a.E, a.k)), 512, 0, s>>>(a);
  decode_down_kernel<W4, NB><<<(a.D + 15) / 16, 512, (size_t)8 * a.T * 16 * 4, s>>>(a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}

}  // namespace sfp8

using namespace sfp8;

extern "C" {

int64_t sfp8_moe_decode_workspace_bytes(int64_t T, int64_t E, int64_t top_k, int64_t I) {
  return decode_sizes_ok(T, E, top_k, 8, I) ? DecodeSpace(T, E, top_k, I).all : -1;
}

int sfp8_moe_decode(const void* x, int64_t ldx, int64_t T, int64_t D, const void* router, int router_type, int64_t E,
                    const void* gate_up, const void* gate_up_scales, const void* down, const void* down_scales,
                    int64_t I, const float* bias, const void* mask, int score, int64_t groups, int64_t top_groups,
                    int64_t group_best, int64_t top_k, int renorm, float scale, int64_t* selected, void* out, void* ws,
                    int64_t ws_bytes, void* stream) {
  if (!decode_sizes_ok(T, E, top_k, D, I) || ldx < 0 || (router_type != kMxF32 && router_type != kMxBf16) ||
      (score != 0 && score != 1) || groups < 1 || groups > 64 || E % groups || top_groups < 1 || top_groups > groups ||
      (group_best != 1 && group_best != 2) || top_k > top_groups * (E / groups) ||
      !gate_up_scales != !down_scales)
    return kErrBadShape;
  if (T == 0) return kOk;
  if (!x || !router || !gate_up || !down || !selected || !out || !ws) return kErrNullPointer;
  const auto off = [](const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) != 0; };
  if (off(x, 2) || off(router, router_type == kMxF32 ? 4 : 2) || off(gate_up, 16) || off(down, 16) ||
      off(gate_up_scales, 4) || off(down_scales, 4) || off(out, 16) || off(ws, 16) || off(selected, 8) || off(bias, 4))
    return kErrBadAlignment;
  const DecodeSpace at(T, E, top_k, I);
  if (ws_bytes < at.all) return kErrWorkspaceTooSmall;
  uint8_t* w = reinterpret_cast<uint8_t*>(ws);
  const DecodeArgs a{(const uint16_t*)x, ldx, (int)T, (int)E, (int)top_k, (int)D, (int)I, router,
                     (int)(router_type == kMxF32), (const uint8_t*)gate_up, (const uint8_t*)gate_up_scales,
                     (const uint8_t*)down, (const uint8_t*)down_scales, bias, (const uint8_t*)mask, score, (int)groups,
                     (int)top_groups, (int)group_best, renorm, scale, selected, (uint16_t*)out, (double*)(w + at.low),
                     (float*)(w + at.weights), (int*)(w + at.plan), (uint16_t*)(w + at.h)};
  const hipStream_t s = (hipStream_t)stream;
  decode_logits_kernel<<<dim3((unsigned)E, (unsigned)((T + kLogitTokens - 1) / kLogitTokens)), 256, 0, s>>>(a);
  // a wave a token, as many as 48 KiB of keys hold
  int waves = T < 16 ? (int)T : 16;
  if (waves > 6144 / E) waves = (int)(6144 / E);
  decode_select_kernel<<<1, 64 * waves, (size_t)waves * E * 8, s>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  const bool one = T <= 16;
  if (gate_up_scales) return one ? launch_experts<true, 1>(a, s) : launch_experts<true, 4>(a, s);
  return one ? launch_experts<false, 1>(a, s) : launch_experts<false, 4>(a, s);
}

}  // extern "C"
