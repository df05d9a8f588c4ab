// A mixture-of-experts layer for a few tokens (gfx950): router, selection,
// gate and up with SwiGLU, down, weighted sum.
//
//   l = x R^T (64-bit sums); the top_k experts and weights as moe_route has
//   them, ordered by values in 64 bits
//   h_j = silu(x Wg_j^T) * (x Wu_j^T);  out = sum_j w_j h_j Wd_j^T
//
// With at most 64 tokens the layer is bound by the bytes of the experts that
// are taken, so their weights are read for all of their tokens at once (down's
// again for each 8 to 32 slots of an expert, from the caches) and go from memory to
// registers (16 bytes a lane); the products run on the bf16 matrix cores with the
// weights as first operand and up to 16 tokens as second.
// Weights are bf16, or MXFP4 codes (mx4.h) that become bf16 values in
// registers, which hold them exactly; x stays bf16 in both.
// Four launches: logits; the selection, a wave a token; gate and up, whose
// work-groups find their expert's slots among all; down and the sum.  Three where
// the router is small (logits and selection in one) and for up to kFused tokens
// (the selection is part of gate and up).
#include <type_traits>

#include "mx4.h"

namespace sfp8 {

constexpr int kMaxTokens = 64, kMaxExperts = 1024, kMaxTopK = 64;
constexpr int kSlots = kMaxTokens * kMaxTopK;  // at most

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
  int* plan;        // per candidate: number of slots (0: not taken); its expert; its slots, 64 each
  float* h;         // [T * k][ldh], zeros from I on
  int ldh;          // I up to a whole number of down's steps
  float* partial;   // [shares of the steps][T, D]
  int* done;        // per column block of down: work-groups that have finished
  int done_count;
};

// Candidates are what may be an expert that is taken: the slots, where they are
// fewer than the experts (a slot stands for its expert if it is the first that
// names it), else the experts.
__host__ __device__ inline int candidates(int T, int E, int k) { return T * k < E ? T * k : E; }
// where the candidates' slots begin in the plan: from 16 bytes on
__host__ __device__ inline int plan_slots(int most) { return (2 * most + 3) / 4 * 4; }

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
// Logits: a work-group takes one expert and TOK tokens, its four waves a quarter
// of the width each.  Sums in 64 bits: products of bf16 with bf16 or fp32 are
// exact in them, and a sum passes at most D / 256 + 8 roundings (a lane's in turn,
// 6 over the lanes, 2 over the waves), so that the order of two experts is that of
// the exact sums but for (D / 256 + 8) 2^-53 of the sum of the products' sizes: 2^-49
// at D = 2048, 2^-41 at the largest.  (A small router's: at most 29 roundings.)
// ---------------------------------------------------------------------------
SFP8_DEV double bf16_at(const Eight<kMxBf16>& v, int j) {
  return (double)__uint_as_float(j & 1 ? v.w[j / 2] & 0xffff0000u : v.w[j / 2] << 16);
}

// N sums over the 64 lanes: a lane hands half of its sums to the lane o away and
// keeps the other half's, then adds over the lanes that hold the same one.  Sum
// n is in the lanes of 64 / N from n on (N = 4: lanes 16 n ..).
template <int N>
SFP8_DEV double lane_sums(double (&v)[N]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int h = N / 2, o = 32; h > 0; h >>= 1, o >>= 1) {
#pragma unroll
    for (int j = 0; j < h; ++j) {
      const double keep = lane & o ? v[j + h] : v[j], give = lane & o ? v[j] : v[j + h];
      v[j] = keep + __shfl_xor(give, o, 64);
    }
  }
#pragma unroll
  for (int o = 32 / N; o > 0; o >>= 1) v[0] += __shfl_xor(v[0], o, 64);
  return v[0];
}

template <int TOK>
__global__ __launch_bounds__(256) void decode_logits_kernel(DecodeArgs a) {
  __shared__ double part[4][TOK];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int e = blockIdx.x, t0 = blockIdx.y * TOK, n = min(TOK, a.T - t0);
  if (e == 0 && t0 == 0)
    for (int i = threadIdx.x; i < a.done_count; i += 256) a.done[i] = 0;
  double acc[TOK];
#pragma unroll
  for (int t = 0; t < TOK; ++t) acc[t] = 0.0;
  for (int d = 8 * threadIdx.x; d < a.D; d += 8 * 256) {
    Eight<kMxBf16> x[TOK];
#pragma unroll
    for (int t = 0; t < TOK; ++t) x[t] = load8<kMxBf16>(a.x, (t0 + min(t, n - 1)) * a.ldx + d);
    double w[8];
    if (a.router_f32) {
      const Eight<kMxF32> v = load8<kMxF32>(a.router, (int64_t)e * a.D + d);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = (double)__uint_as_float(v.w[j]);
    } else {
      const Eight<kMxBf16> v = load8<kMxBf16>(a.router, (int64_t)e * a.D + d);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = bf16_at(v, j);
    }
#pragma unroll
    for (int t = 0; t < TOK; ++t)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[t] = fma(bf16_at(x[t], j), w[j], acc[t]);
  }
  acc[0] = lane_sums<TOK>(acc);
  if (lane % (64 / TOK) == 0) part[wave][lane / (64 / TOK)] = acc[0];
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
  SFP8_DEV double operator()(int e) const { return of(low[e]); }
  SFP8_DEV double of(double l) const { return score == 0 ? exp(l - top) / sum : 1.0 / (1.0 + exp(-l)); }
};

// A wave's choice for token t.  A lane holds the keys of experts lane, lane +
// 64, .. in registers (P of them), so a choice is the maximum of the lanes' best
// (its high words first: seldom do two lanes agree in them) and one lane's
// update.  `shared`: 64 P keys of LDS, read where there are groups.  Afterwards
// lane j has expert and logit of slot j; -1 where nobody is left, and for all
// slots of a masked token.
struct Choice {
  int expert;
  double logit;
};

template <int P>
SFP8_DEV Choice choose(const DecodeArgs& a, int t, const double* low, Scores& s, uint64_t* shared) {
  const int lane = threadIdx.x & 63, E = a.E;
  Choice mine{-1, 0.0};
  s = Scores{low, a.score, 0.0, 1.0};
  if (a.mask && !a.mask[t]) return mine;
  double l[P];
#pragma unroll
  for (int i = 0; i < P; ++i) l[i] = lane + 64 * i < E ? s.low[lane + 64 * i] : -__builtin_inf();
  if (a.score == 0 && (a.bias || (a.groups > 1 && a.group_best == 2) || !a.renorm)) {
    double m = l[0], z = 0.0;
#pragma unroll
    for (int i = 1; i < P; ++i) m = (l[i] > m || l[i] != l[i]) ? l[i] : m;
    s.top = wave_max_or_nan(m);
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (lane + 64 * i < E) z += exp(l[i] - s.top);
    s.sum = wave_sum(z);
  }
  uint64_t key[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int e = lane + 64 * i;
    key[i] = e >= E || l[i] == -__builtin_inf() ? 0 : order_key(a.bias ? s.of(l[i]) + (double)a.bias[e] : l[i]);
  }
  if (a.groups > 1) {
#pragma unroll
    for (int i = 0; i < P; ++i) shared[lane + 64 * i] = key[i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int size = E / a.groups;
    uint64_t best = 0;
    if (lane < a.groups) {
      uint64_t k1 = 0, k2 = 0;
      int e1 = -1, e2 = -1;
      for (int e = lane * size; e < (lane + 1) * size; ++e) {
        const uint64_t x = shared[e];
        if (x > k1) k2 = k1, e2 = e1, k1 = x, e1 = e;
        else if (x > k2) k2 = x, e2 = e;
      }
      best = k1;
      if (a.group_best == 2 && e1 >= 0) {
        double v = s(e1) + (a.bias ? (double)a.bias[e1] : 0.0);
        if (e2 >= 0) v += s(e2) + (a.bias ? (double)a.bias[e2] : 0.0);
        best = order_key(v);
      }
    }
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint64_t other = __shfl(best, g, 64);
      rank += other > best || (other == best && g < lane);
    }
    const uint64_t kept = __ballot(lane < a.groups && best != 0 && rank < a.top_groups);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int e = lane + 64 * i;
      if (e < E && !(kept >> (e / size) & 1)) key[i] = 0;
    }
  }
  for (int j = 0; j < a.k; ++j) {
    uint64_t best = key[0];
    int at = lane;
    double logit = l[0];
#pragma unroll
    for (int i = 1; i < P; ++i)
      if (key[i] > best) best = key[i], at = lane + 64 * i, logit = l[i];
    const uint32_t hi = wave_max_u((uint32_t)(best >> 32));
    bool in = (uint32_t)(best >> 32) == hi;
    uint64_t who = __ballot(in);
    if (who & (who - 1)) {
      const uint32_t lo = wave_max_u(in ? (uint32_t)best : 0u);
      in = in && (uint32_t)best == lo;
      who = __ballot(in);
      if (who & (who - 1)) {  // equals: the lowest index
        const uint32_t first = ~wave_max_u(in ? ~(uint32_t)at : 0u);
        who = __ballot(in && (uint32_t)at == first);
      }
    }
    const int win = __builtin_ctzll(who);
    if (hi == 0 && __builtin_amdgcn_readlane((int)(uint32_t)best, win) == 0) break;  // nobody is left
    const int e = __builtin_amdgcn_readlane(at, win);
    const uint64_t bits = (uint64_t)__double_as_longlong(logit);
    const uint32_t b0 = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, win);
    const uint32_t b1 = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), win);
    if (lane == j) mine = Choice{e, __longlong_as_double((long long)((uint64_t)b1 << 32 | b0))};
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (lane + 64 * i == e) key[i] = 0;
  }
  return mine;
}

// The weights of a wave's choice, shares of the chosen in 64 bits, written with the selection.
SFP8_DEV void write_choice(const DecodeArgs& a, int t, const Scores& s, const Choice& c) {
  const int lane = threadIdx.x & 63;
  const bool there = c.expert >= 0;
  double share;
  if (!a.renorm) {
    share = there ? s.of(c.logit) : 0.0;
  } else {
    // sigmoid(l) = exp(min(l, 0)) / (1 + exp(-|l|)): over exp of the largest min(l, 0) it cannot vanish for all
    const double part = a.score == 0 ? c.logit : (c.logit > 0.0 ? 0.0 : c.logit);
    int width = 1;
    while (width < a.k) width *= 2;
    double m = there ? part : -__builtin_inf();
    for (int o = width / 2; o > 0; o >>= 1) {
      const double w = __shfl_xor(m, o, 64);
      m = (w > m || w != w) ? w : m;
    }
    const double v = exp(part - m);
    share = there ? (a.score == 0 ? v : v / (1.0 + exp(-fabs(c.logit)))) : 0.0;
    double z = share;
    for (int o = width / 2; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
    share /= z;
  }
  if (lane < a.k) {
    a.selected[(int64_t)t * a.k + lane] = c.expert;
    a.weights[t * a.k + lane] = there ? (float)((double)a.scale * share) : 0.f;
  }
}

template <int P>
__global__ __launch_bounds__(64) void decode_select_kernel(DecodeArgs a) {
  __shared__ uint64_t shared[64 * P];
  Scores s;
  const Choice c = choose<P>(a, blockIdx.x, a.low + (int64_t)blockIdx.x * a.E, s, shared);
  write_choice(a, blockIdx.x, s, c);
}

// A small router: a work-group a token has all logits and the selection.  A wave
// takes four experts at a time; where there are fewer than four for each of the
// eight waves, several share the width.  A layer of 16 tokens (us, in a graph): 8
// experts of width 1024 32.5 with it and 33.8 with two kernels, 16 of 512 25.1 and
// 26.1; 16 of 1024 41.0 and 42.0, but 64 of 512 45.1 and 43.9: one CU reads slowly.
constexpr int kSmallRouter = 8192, kSmallExperts = 64;

__global__ __launch_bounds__(512) void decode_router_kernel(DecodeArgs a) {
  constexpr int W = 8;
  __shared__ double part[4 * W], low[kSmallExperts];
  __shared__ uint64_t shared[kSmallExperts];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = blockIdx.x;
  if (t == 0)
    for (int i = threadIdx.x; i < a.done_count; i += 64 * W) a.done[i] = 0;
  const int sets = (a.E + 3) / 4, parts = sets >= W ? 1 : W / sets;
  for (int u = wave; u < sets * parts; u += W) {
    const int e0 = 4 * (u / parts), p = u % parts;
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    for (int d = 8 * (64 * p + lane); d < a.D; d += 512 * parts) {
      const Eight<kMxBf16> x = load8<kMxBf16>(a.x, t * a.ldx + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t at = (int64_t)min(e0 + i, a.E - 1) * a.D + d;
        if (a.router_f32) {
          const Eight<kMxF32> w = load8<kMxF32>(a.router, at);
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[i] = fma(bf16_at(x, j), (double)__uint_as_float(w.w[j]), acc[i]);
        } else {
          const Eight<kMxBf16> w = load8<kMxBf16>(a.router, at);
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[i] = fma(bf16_at(x, j), bf16_at(w, j), acc[i]);
        }
      }
    }
    const double sum = lane_sums<4>(acc);
    if (lane % 16 == 0 && e0 + lane / 16 < a.E) (parts == 1 ? low[e0 + lane / 16] : part[4 * u + lane / 16]) = sum;
  }
  __syncthreads();
  if (parts > 1) {
    for (int e = threadIdx.x; e < a.E; e += 64 * W) {
      double sum = 0.0;
      for (int p = 0; p < parts; ++p) sum += part[4 * (e / 4 * parts + p) + e % 4];
      low[e] = sum;
    }
    __syncthreads();
  }
  if (wave) return;
  Scores s;
  const Choice c = choose<1>(a, t, low, s, shared);
  write_choice(a, t, s, c);
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

// How a lane (row r of 16, quarter q) holds a stretch of K: kStep values of its
// row, of which it has kPieces pieces of 8, piece j at value at(q, j) of the
// stretch.  The four quarters' pieces are neighbours, so that a load's 64 lanes
// read 64 bytes in a run from each of 16 rows; with a lane's own pieces as
// neighbours the first-level cache serves two to four times as many lines.
template <bool W4>
struct Stretch {
  static constexpr int kStep = W4 ? 128 : 64, kPieces = W4 ? 4 : 2;
  static SFP8_DEV int at(int q, int j) { return 32 * j + 8 * q; }
  bf16x8 w[kPieces];
};

// One expert's matrix: at() is a lane's place in row n, `part` stretches further
// on; read() has what the lane holds s stretches from there in flight, values()
// makes bf16 values of it.  Buffer loads: 32-bit offsets from a base in scalar
// registers (a matrix is below 4 GiB), and zeros for what is past its end.
SFP8_DEV __amdgpu_buffer_rsrc_t matrix_rsrc(const uint8_t* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), (short)0, (int)(uint32_t)bytes, 0x00020000);
}
typedef unsigned int uintx4 __attribute__((ext_vector_type(4)));

template <bool W4>
struct WeightRows;
template <>
struct WeightRows<false> {
  using Raw = Stretch<false>;
  struct At {
    uint32_t off;
  };
  __amdgpu_buffer_rsrc_t r;
  uint32_t bytes;  // of a row
  SFP8_DEV WeightRows(const uint8_t* base, const uint8_t*, int64_t e, int64_t rows, int64_t k)
      : r(matrix_rsrc(base + e * rows * k * 2, rows * k * 2)), bytes((uint32_t)k * 2) {}
  SFP8_DEV At at(int n, int part, int q) const { return At{(uint32_t)n * bytes + 128u * part + 16u * q}; }
  SFP8_DEV void read(At at, int s, Raw& f) const {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      f.w[j] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(r, at.off + 128u * s + 64u * j, 0, 0));
  }
  SFP8_DEV void values(const Raw& raw, Stretch<false>& f) const { f = raw; }
  // what is past column K, the next row's, as zeros; k: the stretch's first column
  static SFP8_DEV void zero_past(Stretch<false>& f, int K, int k, int q) {
#pragma unroll
    for (int j = 0; j < 2; ++j) f.w[j] = zero_unless(k + Stretch<false>::at(q, j) < K, f.w[j]);
  }
};
template <>
struct WeightRows<true> {
  struct Raw {
    uintx4 codes;
    uint32_t scales;
  };
  struct At {
    uint32_t row;
    uint32_t q;
  };
  __amdgpu_buffer_rsrc_t r, rs;  // [slabs][rows rounded up][64], [..][4]
  uint32_t rows;
  SFP8_DEV WeightRows(const uint8_t* c, const uint8_t* s, int64_t e, int64_t n, int64_t k)
      : r(matrix_rsrc(c + e * mx_slabs(k) * mx_rows(n) * 64, mx_slabs(k) * mx_rows(n) * 64)),
        rs(matrix_rsrc(s + e * mx_slabs(k) * mx_rows(n) * 4, mx_slabs(k) * mx_rows(n) * 4)),
        rows((uint32_t)mx_rows(n)) {}
  SFP8_DEV At at(int n, int part, int q) const { return At{(uint32_t)part * rows + n, 16u * q}; }
  SFP8_DEV void read(At at, int s, Raw& f) const {
    const uint32_t row = at.row + (uint32_t)s * rows;
    f.codes = __builtin_amdgcn_raw_buffer_load_b128(r, row * 64 + at.q, 0, 0);
    f.scales = __builtin_amdgcn_raw_buffer_load_b32(rs, row * 4, 0, 0);
  }
  // A lane has read block q of the row; piece j is a quarter of block j: a transpose of the quarters' words.
  SFP8_DEV void values(const Raw& raw, Stretch<true>& f) const {
    const auto a = __builtin_amdgcn_permlane32_swap(raw.codes[0], raw.codes[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(raw.codes[1], raw.codes[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    const uint32_t word[4] = {c[0], c[1], d[0], d[1]};
#pragma unroll
    for (int j = 0; j < 4; ++j) f.w[j] = bf16_of_codes8(word[j], mx_scale_value(raw.scales >> (8 * j) & 255u));
  }
  static SFP8_DEV void zero_past(Stretch<true>&, int, int, int) {}  // padding has zero codes, past the end are zeros
};

// A token's values beside them; `row` is the lane's own place, 8 q values into the row.
template <bool W4>
SFP8_DEV void read_values(const uint16_t* row, int k, Stretch<W4>& f) {
#pragma unroll
  for (int j = 0; j < Stretch<W4>::kPieces; ++j) f.w[j] = load_bf16x8(row + k + 32 * j);
}
// ... of a stretch that the row ends in: zeros from column K (a multiple of 8) on.
template <bool W4>
SFP8_DEV void read_last(const uint16_t* row, int K, int k, int q, Stretch<W4>& f) {
#pragma unroll
  for (int j = 0; j < Stretch<W4>::kPieces; ++j) {
    const int at = k + Stretch<W4>::at(q, j);
    f.w[j] = zero_unless(at < K, load_bf16x8(row + (at < K ? at : K - 8) - 8 * q));
  }
}

// Four values of h as three bf16 values each: the upper eight bits of what is
// left, three times, are all 24 of a value (down to bf16's smallest), and the
// products of bf16 values are exact, so the sums are those of h in 32 bits.  An
// infinity leaves nothing.
SFP8_DEV void three_parts(const intx4& v, intx2 (&part)[3]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t left[2] = {(uint32_t)v[2 * i], (uint32_t)v[2 * i + 1]};
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      part[p][i] = (int)__builtin_amdgcn_perm(left[1], left[0], 0x07060302u);
      if (p < 2) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float f = __uint_as_float(left[j]);
          const float rest = f - __uint_as_float(left[j] & 0xffff0000u);
          left[j] = p == 0 && !__builtin_isfinite(f) ? 0u : __float_as_uint(rest);
        }
      }
    }
  }
}

// n steps as calls of f(size, first) with sizes U, U / 2, .., 1 (compile-time).
template <int U, class F>
SFP8_DEV void in_batches(int n, F f, int i = 0) {
  for (; i + U <= n; i += U) f(std::integral_constant<int, U>{}, i);
  if constexpr (U > 1) in_batches<U / 2>(n, f, i);
}

// Up to this many tokens are selected by the waves of every work-group of gate
// and up (P keys a lane): 3 us that it waits longer against 6 of a launch and a
// kernel of its own.  (Layer in a graph, us: one token, 8 of 128 experts, bf16 28.3
// against 32.3, 4-bit 19.9 against 22.2; four tokens, 2 of 128, 18.9 against 21.0.)
constexpr int kFused = 4, kFusedKeys = 4, kFusedGroups = 1024;

// Gate and up of 8 columns of h for all slots of one expert: a product's 16 rows
// are the 8 gate rows and the 8 up rows.  Four waves share the width, up to four
// steps of each in flight, and their sums meet in LDS in the order of the waves.
// Small work-groups, several a CU: with one token and eight experts of 768
// columns there are three for each CU, and their waits overlap.  NB: blocks of
// 16 slots that an expert can have.
template <bool W4, int NB, int SETS>
__global__ __launch_bounds__(256, W4 && NB > 1 ? 3 : 4) void decode_gateup_kernel(DecodeArgs a) {
  constexpr int W = 4, kStep = Stretch<W4>::kStep, kPieces = Stretch<W4>::kPieces;
  constexpr bool FUSED = SETS == 1;
  static_assert(!FUSED || (kFused <= W && NB == 1), "a wave a token");
  __shared__ __align__(16) float red[W][SETS][16][20];
  __shared__ int list[kMaxTokens], count[W], own;
  __shared__ uint64_t keys[FUSED ? W * 64 * kFusedKeys : 1];
  __shared__ short chosen[FUSED ? kFused * kMaxTopK : 1];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // the expert of this candidate, and its slots in order
  const int slots = a.T * a.k, most = candidates(a.T, a.E, a.k), c = blockIdx.y;
  if constexpr (FUSED) {
    if (c == most && blockIdx.x) return;  // one work-group more writes the selection and the weights
    if (wave < a.T) {
      Scores s;
      const Choice x = choose<kFusedKeys>(a, wave, a.low + (int64_t)wave * a.E, s, keys + wave * 64 * kFusedKeys);
      if (c == most) write_choice(a, wave, s, x);
      else if (lane < a.k) chosen[wave * a.k + lane] = (short)x.expert;
    }
    if (c == most) return;
    __syncthreads();
  }
  const auto expert_of = [&](int s) { return FUSED ? (int)chosen[FUSED ? s : 0] : (int)a.selected[s]; };
  const bool by_slot = slots < a.E;
  int e = c, n = 0;
  for (int s0 = 0; s0 < slots; s0 += 64 * W) {
    const int s = s0 + tid, x = s < slots ? expert_of(s) : -1;
    if (by_slot && s0 == 0) {
      if (c < 64 * W ? s == c : tid == 0) own = c < 64 * W ? x : expert_of(c);
      __syncthreads();
      e = own;
    }
    const bool match = e >= 0 && x == e;
    const uint64_t who = __ballot(match);
    if (lane == 0) count[wave] = __builtin_popcountll(who);
    __syncthreads();
    int before = n;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < wave) before += count[w];
      n += count[w];
    }
    if (match) list[before + __builtin_popcountll(who & ((1ull << lane) - 1))] = s;
    __syncthreads();
  }
  if (by_slot && n > 0 && list[0] != c) n = 0;  // an earlier slot stands for this expert
  if (blockIdx.x == 0) {
    if (tid == 0) a.plan[c] = n, a.plan[most + c] = e;
    if (tid < n) a.plan[plan_slots(most) + 64 * c + tid] = list[tid];
  }
  if (n == 0) return;

  e = __builtin_amdgcn_readfirstlane(e);
  n = __builtin_amdgcn_readfirstlane(n);
  const int i0 = 8 * SETS * blockIdx.x, D = a.D, I = a.I;  // I is a multiple of 8
  const WeightRows<W4> w(a.gu, a.gu_scales, e, 2 * (int64_t)I, D);
  typename WeightRows<W4>::At row[SETS];
#pragma unroll
  for (int z = 0; z < SETS; ++z) row[z] = w.at((r < 8 ? 0 : I - 8) + r + min(i0 + 8 * z, I - 8), 0, q);
  const uint16_t* xrow[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int s = 16 * b + r;  // a lane without a slot goes along with the first
    xrow[b] = a.x + (list[s < n ? s : 0] / a.k) * a.ldx + 8 * q;
  }
  floatx4 acc[NB][SETS];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int z = 0; z < SETS; ++z) acc[b][z] = floatx4{0.f, 0.f, 0.f, 0.f};
  const auto multiply = [&](const Stretch<W4> (&fw)[SETS], const Stretch<W4>& fx, int b) {
#pragma unroll
    for (int z = 0; z < SETS; ++z)
#pragma unroll
      for (int j = 0; j < kPieces; ++j) acc[b][z] = mfma16(fw[z].w[j], fx.w[j], acc[b][z]);
  };
  const int full = D / kStep;
  const auto batch = [&](auto size, int s) {  // steps s, s + W, ..: all of their bytes in flight at once
    constexpr int U = decltype(size)::value;
    typename WeightRows<W4>::Raw raw[U][SETS];
    Stretch<W4> fx[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
#pragma unroll
      for (int z = 0; z < SETS; ++z) w.read(row[z], s + i * W, raw[i][z]);
      read_values<W4>(xrow[0], (s + i * W) * kStep, fx[i]);
    }
    __builtin_amdgcn_sched_barrier(0);  // the loads stay ahead of the products
#pragma unroll
    for (int i = 0; i < U; ++i) {
      Stretch<W4> fw[SETS];
#pragma unroll
      for (int z = 0; z < SETS; ++z) w.values(raw[i][z], fw[z]);
      multiply(fw, fx[i], 0);
#pragma unroll
      for (int b = 1; b < NB; ++b) {
        if (16 * b < n) {
          Stretch<W4> more;
          read_values<W4>(xrow[b], (s + i * W) * kStep, more);
          multiply(fw, more, b);
        }
      }
    }
  };
  constexpr int kMost = SETS > 1 && (W4 || NB > 1) ? 2 : 4;  // what the registers of four waves a SIMD hold
  in_batches<kMost>((full - wave + W - 1) / W, [&](auto size, int i) { batch(size, wave + i * W); });
  if (D % kStep && wave == full % W) {
    typename WeightRows<W4>::Raw raw;
    Stretch<W4> fw[SETS], fx;
#pragma unroll
    for (int z = 0; z < SETS; ++z) {
      w.read(row[z], full, raw);
      w.values(raw, fw[z]);
      w.zero_past(fw[z], D, full * kStep, q);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if (16 * b < n) {
        read_last<W4>(xrow[b], D, full * kStep, q, fx);
        multiply(fw, fx, b);
      }
    }
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    if (16 * b >= n) break;
    if (b) __syncthreads();
#pragma unroll
    for (int z = 0; z < SETS; ++z) *reinterpret_cast<floatx4*>(&red[wave][z][r][4 * q]) = acc[b][z];
    __syncthreads();
    const int s = tid / (8 * SETS), col = tid % (8 * SETS), z = col >> 3;
    if (s < 16 && 16 * b + s < n && i0 + col < I) {
      float g = 0.f, u = 0.f;
#pragma unroll
      for (int v = 0; v < W; ++v) g += red[v][z][s][col & 7], u += red[v][z][s][8 + (col & 7)];
      // exp's argument is not rounded first, as exp2 of g log2(e) would have it: that is off by |g| / 2 steps
      a.h[(int64_t)list[16 * b + s] * a.ldh + i0 + col] = g / (1.f + expf(-g)) * u;
    }
  }
  if (i0 + 8 * SETS >= I && a.ldh > I) {  // zeros up to the end of down's last stretch
    const int pad = a.ldh - I;
    for (int i = tid; i < n * pad; i += 64 * W) a.h[(int64_t)list[i / pad] * a.ldh + I + i % pad] = 0.f;
  }
}

// Down and the weighted sum for C SETS columns of the output: the steps of all
// experts that are taken are dealt out to the waves in even runs.  A wave adds
// each expert's sums times the slots' weights to its own totals of all tokens
// (LDS), and the waves' totals meet in their order: no sum depends on the order of
// arrival.
// A product's 16 rows are C columns in P = 16 / C parts of K, its 16 columns C
// slots in the same parts, and of the result the blocks where the parts agree
// are kept: a CU takes no more than about 20 bytes a nanosecond from memory, so
// all of them have to have a work-group.  An expert of more than 2 C slots is
// read again for each 2 C of them.  RAGGED: I is no multiple of a step.
// h is in 32 bits.  A wave reads each value of a step once (16 lanes 64 columns
// of a slot and part), splits it into three bf16 parts and hands them to the
// matrix cores' lanes through its own LDS.  Where the slots take a quarter of the
// product's columns at most, their parts are columns of their own: a third of the
// LDS reads and products, and the three sums meet at the end.  (Layer of 2048 x
// 768, 8 of 128 experts, in a graph, us: 4 tokens 4-bit 38.8, 16 tokens bf16 158.5;
// every lane splitting what it multiplies, without LDS, 46.6 and 172; h in two
// bf16 parts as they lie in memory, 17 bits of it, 38.4 and 168.)
// With many slots an expert, h is what the CUs take most of (32 bits of each
// slot beside C rows of weights): then SETS = 2 sets of 16 columns share it, and
// gridDim.y work-groups share the steps of a column block; the last of them to
// finish (counters that the logits' launch has zeroed) adds their sums in order.
template <bool W4, int C, int SETS, bool RAGGED>
__global__ __launch_bounds__(512) void decode_down_kernel(DecodeArgs a) {
  static_assert(SETS == 1 || C == 16, "");
  constexpr int W = 8, P = 16 / C, CB = C * SETS, NB = 2;
  constexpr int kStep = P * Stretch<W4>::kStep, kSubs = Stretch<W4>::kPieces / 2;
  // rows of 64 bf16 values, 16 bytes further on by the banks from one to the next
  constexpr int kHRow = 144, kMostTogether = SETS > 1 ? 1 : kSubs;  // 64 columns a unit
  extern __shared__ __align__(16) float totals[];  // [W][T][CB]
  __shared__ __align__(16) uint8_t hparts[W][kMostTogether * 3 * 16 * kHRow];
  __shared__ short expert_of[kMaxExperts], slot_of[kSlots];
  __shared__ int begin[kMaxExperts + 1], count[W], slots_before[W], last;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = CB * blockIdx.x, D = a.D, I = a.I, T = a.T, most = candidates(T, a.E, a.k);
  float* mine = totals + wave * T * CB;
  uint8_t* hs = hparts[wave];
  for (int i = lane; i < T * CB / 4; i += 64) reinterpret_cast<floatx4*>(mine)[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  // the experts that are taken, in the candidates' order, and their slots
  int live = 0, taken = 0;
  for (int c0 = 0; c0 < most; c0 += 64 * W) {
    const int c = c0 + tid;
    const int* list = a.plan + plan_slots(most) + 64 * c;
    int n = 0, e = 0, some[4];
    if (c < most) {  // all at once: the list's first slots whether there or not
      n = a.plan[c], e = a.plan[most + c];
      const intx4 v = *reinterpret_cast<const intx4*>(list);
#pragma unroll
      for (int i = 0; i < 4; ++i) some[i] = v[i];
    }
    const uint64_t who = __ballot(n > 0);
    int upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int p = __shfl_up(upto, o, 64);
      if (lane >= o) upto += p;
    }
    if (lane == 63) count[wave] = __builtin_popcountll(who), slots_before[wave] = upto;
    __syncthreads();
    int at = live + __builtin_popcountll(who & ((1ull << lane) - 1)), first = taken + upto - n;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < wave) at += count[w], first += slots_before[w];
      live += count[w], taken += slots_before[w];
    }
    if (n > 0) {
      expert_of[at] = (short)e;
      begin[at] = first;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < n) slot_of[first + i] = (short)some[i];
      for (int i = 4; i < n; ++i) slot_of[first + i] = (short)list[i];
    }
    __syncthreads();
  }
  if (tid == 0) begin[live] = taken;
  __syncthreads();
  const int steps = (I + kStep - 1) / kStep;
  const int64_t all = (int64_t)live * steps;
  const int turn = blockIdx.y * W + wave, turns = gridDim.y * W;
  const int lo = (int)(all * turn / turns), hi = (int)(all * (turn + 1) / turns);
  const int part = r / C;
  for (int at = lo; at < hi;) {
    const int which = at / steps, s0 = at - which * steps, s1 = min(steps, s0 + hi - at);
    at += s1 - s0;
    const int end = __builtin_amdgcn_readfirstlane(begin[which + 1]);
    const WeightRows<W4> w(a.down, a.down_scales, __builtin_amdgcn_readfirstlane(expert_of[which]), D, I);
    typename WeightRows<W4>::At place[SETS];
#pragma unroll
    for (int z = 0; z < SETS; ++z) place[z] = w.at(min(n0 + C * z + r % C, D - 1), part, q);
    for (int first = __builtin_amdgcn_readfirstlane(begin[which]); first < end; first += NB * C) {
      const int n = min(end - first, NB * C);
      const auto products = [&](auto blocks, auto loads) {
        constexpr int B = decltype(blocks)::value, X = decltype(loads)::value;
        constexpr int kRegs = SETS * (int)sizeof(typename WeightRows<W4>::Raw) / 4 + B * kSubs * X * 4;
        // slots that are few enough have their parts in columns of their own: one product in the place of three, and
        // three steps a way through the LDS
        constexpr bool kApart = X == 1;
        constexpr int kParts = kApart ? 1 : 3, kTogether = kApart ? kSubs : kMostTogether;
        constexpr int kSteps = kApart ? 3 * kMostTogether / kSubs : 1;
        constexpr int kUnitRows = 16 * kParts, kPartRows = kApart ? 1 : 16;
        // Steps in flight: three, or as many as 256 registers hold.  Up to eight are 49 KB of code in the place of 25 -
        // 33, which each launch fetches anew (4 tokens 4-bit 40.2 us against 38.8, 16 tokens bf16 160.7, 158.5).
        constexpr int kSpace = SETS > 1 ? 112 : kMostTogether > 1 ? 128 : 160;
        constexpr int kInFlight = kSpace / kRegs < 3 ? kSpace / kRegs : 3;
        const float* hrow[B][X];
        uint32_t to[X];
#pragma unroll
        for (int x = 0; x < X; ++x) {
          const int u = 4 * x + q, slot = u / P, prt = u % P;
          to[x] = (uint32_t)(prt * C + (kApart ? 3 * slot : slot)) * kHRow + 8 * r;
#pragma unroll
          for (int b = 0; b < B; ++b) {
            const int i = C * b + slot;
            hrow[b][x] = a.h + (int64_t)slot_of[first + (i < n ? i : 0)] * a.ldh + prt * Stretch<W4>::kStep + 4 * r;
          }
        }
        const auto slot_in = [&](int b) { return kApart ? r % C / 3 : C * b + r % C; };  // that this lane's sums are of
        float weight[B];
#pragma unroll
        for (int b = 0; b < B; ++b) weight[b] = a.weights[slot_of[first + (slot_in(b) < n ? slot_in(b) : 0)]];
        floatx4 acc[B][SETS];
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
          for (int z = 0; z < SETS; ++z) acc[b][z] = floatx4{0.f, 0.f, 0.f, 0.f};
        in_batches<kInFlight>(s1 - s0, [&](auto size, int from) {
          constexpr int U = decltype(size)::value;
          typename WeightRows<W4>::Raw rw[U][SETS];
          intx4 f[U][B][kSubs][X];
#pragma unroll
          for (int i = 0; i < U; ++i) {
            const int s = s0 + from + i;
#pragma unroll
            for (int z = 0; z < SETS; ++z) w.read(place[z], P * s, rw[i][z]);
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
              for (int u = 0; u < kSubs; ++u)
#pragma unroll
                for (int x = 0; x < X; ++x)
                  f[i][b][u][x] = *reinterpret_cast<const intx4*>(hrow[b][x] + s * kStep + 64 * u);
          }
          __builtin_amdgcn_sched_barrier(0);  // the loads stay ahead of the products
          Stretch<W4> fw[SETS];
          const auto weights = [&](int i) {
            const int s = s0 + from + i;
#pragma unroll
            for (int z = 0; z < SETS; ++z) {
              w.values(rw[i][z], fw[z]);
              if (RAGGED && s == steps - 1) w.zero_past(fw[z], I, s * kStep + part * Stretch<W4>::kStep, q);
            }
          };
#pragma unroll
          for (int i0 = 0; i0 < U; i0 += kSteps) {
            if constexpr (kSteps == 1) weights(i0);
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
              for (int u0 = 0; u0 < kSubs; u0 += kTogether) {
#pragma unroll
                for (int c = 0; c < kSteps && i0 + c < U; ++c)
#pragma unroll
                  for (int u = 0; u < kTogether; ++u)
#pragma unroll
                    for (int x = 0; x < X; ++x) {
                      intx2 h[3];
                      three_parts(f[i0 + c][b][u0 + u][x], h);
#pragma unroll
                      for (int p = 0; p < 3; ++p)
                        *reinterpret_cast<intx2*>(hs + ((c * kTogether + u) * kUnitRows + p * kPartRows) * kHRow +
                                                  to[x]) = h[p];
                    }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                bf16x8 h[kSteps][kTogether][2][kParts];
#pragma unroll
                for (int c = 0; c < kSteps && i0 + c < U; ++c)
#pragma unroll
                  for (int u = 0; u < kTogether; ++u)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                      for (int p = 0; p < kParts; ++p)
                        h[c][u][j][p] = *reinterpret_cast<const bf16x8*>(
                            hs + ((c * kTogether + u) * kUnitRows + p * 16 + r) * kHRow + 64 * j + 16 * q);
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
                for (int c = 0; c < kSteps && i0 + c < U; ++c) {
                  if constexpr (kSteps > 1) weights(i0 + c);
#pragma unroll
                  for (int u = 0; u < kTogether; ++u)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                      for (int p = 0; p < kParts; ++p)
#pragma unroll
                        for (int z = 0; z < SETS; ++z)
                          acc[b][z] = mfma16(fw[z].w[2 * (u0 + u) + j], h[c][u][j][p], acc[b][z]);
                }
              }
          }
        });
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
          for (int z = 0; z < SETS; ++z) {
            floatx4 v = acc[b][z];
            // a part's columns are 4 q' .. + 3 of slot r % C: the next part's lie 256 / P + C lanes on (rows, columns)
            if constexpr (P > 1) {
              floatx4 sum = v;
#pragma unroll
              for (int o = 1; o < P; ++o)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] += __shfl(v[j], (lane + o * (64 / P + C)) & 63, 64);
              v = sum;
            }
            if constexpr (kApart) {
#pragma unroll
              for (int j = 0; j < 4; ++j) v[j] += __shfl(v[j], (lane + 1) & 63, 64) + __shfl(v[j], (lane + 2) & 63, 64);
            }
            if (slot_in(b) < n && (!kApart || r % 3 == 0) && r < C && q < C / 4) {
              floatx4* p = reinterpret_cast<floatx4*>(mine + slot_of[first + slot_in(b)] / a.k * CB + C * z + 4 * q);
              floatx4 t = *p;
#pragma unroll
              for (int j = 0; j < 4; ++j) t[j] = __builtin_fmaf(weight[b], v[j], t[j]);
              *p = t;
            }
          }
      };
      const auto one = std::integral_constant<int, 1>{};
      if (n > C) products(std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
      else if (P * n > 8) products(one, std::integral_constant<int, 4>{});
      else if (P * n > 4) products(one, std::integral_constant<int, 2>{});
      else products(one, one);
    }
  }
  __syncthreads();
  const bool shared = gridDim.y > 1;
  for (int i = tid; i < T * CB / 2; i += 64 * W) {
    const int t = i / (CB / 2), col = 2 * (i % (CB / 2));
    float v0 = 0.f, v1 = 0.f;
#pragma unroll
    for (int v = 0; v < W; ++v) v0 += totals[(v * T + t) * CB + col], v1 += totals[(v * T + t) * CB + col + 1];
    if (n0 + col < D) {
      const int64_t at = (int64_t)t * D + n0 + col;
      if (shared) *reinterpret_cast<floatx2*>(a.partial + (int64_t)blockIdx.y * T * D + at) = floatx2{v0, v1};
      else *reinterpret_cast<uint32_t*>(a.out + at) = pack2_bf16(v0, v1);
    }
  }
  if (!shared) return;
  // Every wave's sums are in the L2 before the barrier (which by itself waits for none); thread 0's release and acquire
  // then work on the whole L2 and on this CU's cache.  Done by every wave they took as long as the products.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0)
    last = __hip_atomic_fetch_add(a.done + blockIdx.x, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
           (int)gridDim.y - 1;
  __syncthreads();
  if (!last) return;
  for (int i = tid; i < T * CB / 2; i += 64 * W) {
    const int t = i / (CB / 2), col = 2 * (i % (CB / 2));
    if (n0 + col < D) {
      const int64_t at = (int64_t)t * D + n0 + col;
      floatx2 v = {0.f, 0.f};
      for (int y = 0; y < (int)gridDim.y; ++y) {
        const floatx2 p = *reinterpret_cast<const floatx2*>(a.partial + (int64_t)y * T * D + at);
        v[0] += p[0], v[1] += p[1];
      }
      *reinterpret_cast<uint32_t*>(a.out + at) = pack2_bf16(v[0], v[1]);
    }
  }
}

inline int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

// work-groups that share the steps of a block of 32 columns (T > 16): about one for each CU in all
inline int down_shares(int64_t T, int64_t D) {
  const int64_t blocks = (D + 31) / 32;
  return T <= 16 || blocks >= 256 ? 1 : (int)(blocks <= 16 ? 16 : 256 / blocks);
}

struct DecodeSpace {
  int64_t low, weights, plan, done, partial, h, all;
  DecodeSpace(int64_t T, int64_t E, int64_t k, int64_t D, int64_t I) {
    const int64_t most = candidates((int)T, (int)E, (int)k), shares = down_shares(T, D);
    low = 0;
    weights = low + up256(T * E * 8);
    plan = weights + up256(T * k * 4);
    done = plan + up256((plan_slots((int)most) + 64 * most) * 4);
    partial = done + up256(shares > 1 ? (D + 31) / 32 * 4 : 0);
    h = partial + up256(shares > 1 ? shares * T * D * 4 : 0);
    all = h + T * k * ((I + 511) / 512 * 512) * 4;  // a step of down has at most 512 columns
  }
};

inline bool decode_sizes_ok(int64_t T, int64_t E, int64_t k, int64_t D, int64_t I) {
  return T >= 0 && T <= kMaxTokens && E >= 1 && E <= kMaxExperts && k >= 1 && k <= kMaxTopK && k <= E && D >= 8 &&
         D % 8 == 0 && D <= 1 << 20 && I >= 8 && I % 8 == 0 && I <= 1 << 20 && D * I <= (int64_t)1 << 29;
}

template <bool W4, int C, int SETS>
void launch_down(const DecodeArgs& a, int shares, hipStream_t s) {
  const dim3 grid((unsigned)((a.D + C * SETS - 1) / (C * SETS)), (unsigned)shares);
  const size_t totals = (size_t)8 * a.T * C * SETS * 4;
  if (a.I != a.ldh) decode_down_kernel<W4, C, SETS, true><<<grid, 512, totals, s>>>(a);
  else decode_down_kernel<W4, C, SETS, false><<<grid, 512, totals, s>>>(a);
}

template <bool W4>
void launch_experts(DecodeArgs a, hipStream_t s) {
  // Columns a work-group of down: such that at D = 1024 (bf16), 2048 and 4096 there is one for each CU; narrower layers
  // leave CUs without one.  In a graph, us a layer with 4, 8 and 16 columns:
  //  bf16  T = 16, D = 1024, 2 of 8 experts of 1536 32.9, 34.1, 37.9; T = 4, D = 512, the same ones 21.3, 22.7, 26.8;
  //        T = 1, D = 2048, 8 of 128 of 768 31.5, 27.8, 30.6; T = 4, D = 4096, 2 of 16 of 1536 73.3, 63.8, 60.0
  //  4-bit T = 4, 8 of 128 of 768, D = 512 30.0, 31.9, 37.3; 1024 34.1, 35.2, 40.3; 2048 50.8, 40.1, 45.3; D = 4096, 8
  //        of 32 77.7, 55.9, 48.1
  // Beyond 16 tokens 32 columns, whose steps are shared (T = 64, D = 2048, 6 of 64 of 1032: 185 against 227 with 16;
  // T = 24, D = 1024, 2 of 8: 35.5 against 42.3; T = 16, the first of the layers above: 33.8).
  const int C = a.T > 16 ? 32 : a.D >= 4096 ? 16 : !W4 && a.D < 2048 ? 4 : 8;
  const int step = (C < 16 ? 16 / C : 1) * Stretch<W4>::kStep;
  a.ldh = (a.I + step - 1) / step * step;
  const unsigned most = (unsigned)candidates(a.T, a.E, a.k);
  const bool fused = a.T <= kFused && a.E <= 64 * kFusedKeys && most * (unsigned)(a.I / 8) <= kFusedGroups;
  const bool small = !fused && a.E <= kSmallExperts && a.E * a.D <= kSmallRouter;
  if (small) decode_router_kernel<<<a.T, 512, 0, s>>>(a);
  else if (a.T == 1) decode_logits_kernel<1><<<dim3(a.E, 1), 256, 0, s>>>(a);
  else decode_logits_kernel<4><<<dim3(a.E, (a.T + 3) / 4), 256, 0, s>>>(a);
  if (fused) {
    decode_gateup_kernel<W4, 1, 1><<<dim3((unsigned)(a.I / 8), most + 1), 256, 0, s>>>(a);
  } else {
    if (!small) {
      if (a.E <= 256) decode_select_kernel<4><<<a.T, 64, 0, s>>>(a);
      else decode_select_kernel<16><<<a.T, 64, 0, s>>>(a);
    }
    const dim3 grid((unsigned)((a.I + 15) / 16), most);
    if (a.T <= 16) decode_gateup_kernel<W4, 1, 2><<<grid, 256, 0, s>>>(a);
    else decode_gateup_kernel<W4, 4, 2><<<grid, 256, 0, s>>>(a);
  }
  if (C == 32) launch_down<W4, 16, 2>(a, down_shares(a.T, a.D), s);
  else if (C == 16) launch_down<W4, 16, 1>(a, 1, s);
  else if (W4 || C == 8) launch_down<W4, 8, 1>(a, 1, s);
  else if constexpr (!W4) launch_down<W4, 4, 1>(a, 1, s);
}

}  // namespace sfp8

using namespace sfp8;

extern "C" {

int64_t sfp8_moe_decode_workspace_bytes(int64_t T, int64_t E, int64_t top_k, int64_t D, int64_t I) {
  return decode_sizes_ok(T, E, top_k, D, I) ? DecodeSpace(T, E, top_k, D, I).all : -1;
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
  const DecodeSpace at(T, E, top_k, D, I);
  if (ws_bytes < at.all) return kErrWorkspaceTooSmall;
  uint8_t* w = reinterpret_cast<uint8_t*>(ws);
  const DecodeArgs a{(const uint16_t*)x, ldx, (int)T, (int)E, (int)top_k, (int)D, (int)I, router,
                     (int)(router_type == kMxF32), (const uint8_t*)gate_up, (const uint8_t*)gate_up_scales,
                     (const uint8_t*)down, (const uint8_t*)down_scales, bias, (const uint8_t*)mask, score, (int)groups,
                     (int)top_groups, (int)group_best, renorm, scale, selected, (uint16_t*)out, (double*)(w + at.low),
                     (float*)(w + at.weights), (int*)(w + at.plan), (float*)(w + at.h), 0,
                     (float*)(w + at.partial), (int*)(w + at.done),
                     down_shares(T, D) > 1 ? (int)((D + 31) / 32) : 0};
  const hipStream_t s = (hipStream_t)stream;
  if (gate_up_scales) launch_experts<true>(a, s);
  else launch_experts<false>(a, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? kOk : (int)e;
}

}  // extern "C"
