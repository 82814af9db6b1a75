// A row's log probabilities and entropy from sums about its largest logit, shared by
// the operators that give them.
//
// With M the largest logit, n logits alike to it and y_j = a (z_j - M) log2(e) <= 0:
//   S = sum 2^y = n + S',  T = sum y 2^y = T'      (S', T': over the others)
//   log q_j = ln 2 (y_j - log2 S),   H = -sum q log q = ln 2 (log2 S - T / S)
// Both terms of H are positive, and S' is summed without the n: a token of
// probability 1 - 1e-9 has log q = -log1p(S') and H to the sums' own rounding (as
// 1 + S' in 32 bits both would be 0). Sums of a wave are in 32 bits, and joined, with
// all that follows, in 64: with alternatives the kernel is bound by its instructions, and a
// 64-bit exponential would be a dozen for one. What that costs: 4e-8 of the outputs' size
// where sums in 64 bits leave 3e-8 (2039 x 65536 bf16, the rounding to float32 included),
// 5e-8 for 2e-8 to 5e-8 in one row.
#pragma once

#include "logits_rows.h"

namespace rwkv7 {

constexpr double kLn2 = 0.69314718055994531;

// log(n + s), n >= 1, s >= 0, to 1e-11 of itself.
RWKV7_DEV double log_n_plus(double n, double s) {
  if (n == 1.0 && s < 0.03125)  // the logarithm's own series: s^8 / 9 of it is left out
    return s * (1.0 - s * (0.5 - s * (1.0 / 3 - s * (0.25 - s * (0.2 - s * (1.0 / 6 - s * (1.0 / 7 - s * 0.125)))))));
  return kLn2 * log2_d(n + s);
}
// 1 - exp(y), y <= 0, to 1e-10 of itself.
RWKV7_DEV double one_minus_exp(double y) {
  if (y > -0.03125)  // the exponential's own series: y^6 / 5040 of it is left out
    return -y * (1.0 + y * (0.5 + y * (1.0 / 6 + y * (1.0 / 24 + y * (1.0 / 120 + y * (1.0 / 720))))));
  return 1.0 - (y == y ? exp2_d(1.4426950408889634 * y) : y);
}

// RowMax by halves in pairs for bfloat16 too, as whole numbers: the largest of these is
// the largest logit where one is positive, and else the least is. Where a NaN that
// counts as positive is among them it is not, and the caller takes RowMax.
template <int FMT>
struct PairMax : RowMax<FMT> {
  RWKV7_DEV bool clean() const { return true; }
};
template <>
struct PairMax<2> {
  typedef short short2v __attribute__((ext_vector_type(2)));
  short2v most = {-32768, -32768}, least = {32767, 32767};
  RWKV7_DEV void add(const Chunk<2> &x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const short2v v = __builtin_bit_cast(short2v, x.w[i]);
      most = __builtin_elementwise_max(most, v);
      least = __builtin_elementwise_min(least, v);
    }
  }
  RWKV7_DEV bool clean() const { return max(most[0], most[1]) <= 0x7f80; }
  RWKV7_DEV float value() const {
    const short m = max(most[0], most[1]), l = min(least[0], least[1]);
    return m >= 0 ? b2f((uint16_t)m) : l > -128 ? -kInf : b2f((uint16_t)l);  // (0xff80 is -inf; NaN beyond)
  }
};

struct ScoreLds {
  float m[kMaxWaves], S[kMaxWaves], T[kMaxWaves];
  int n[kMaxWaves];
};

// What the waves have of the row: S', T' and n about M as score_arg() forms the exponents,
// which lie `at` (their own value at M) above y.
struct RowSums {
  double S, T, n, at;
  double slope;  // ln 2 times what log2(e) / temperature has over its float, of itself
  float M;
};

// The exponent of an element, and of M (ref: M, or 0 for none), in 32 bits.
RWKV7_DEV float near_arg(const ExpScale &sc, float x, float ref) { return fmaf(x, sc.kf, -(ref * sc.kf)); }
RWKV7_DEV float score_arg(const ExpScale &sc, float x, float ref) {
  return sc.near(ref) ? near_arg(sc, x, ref) : (x - ref) * sc.kf;
}

// Sums of a wave's row about M (wave-uniform, the largest of all waves, `own` this
// wave's largest). A NaN among the logits makes S NaN; M is the largest of the others.
// Where a logit is masked, T comes out NaN by 0 times -inf: then, and far from 0 (see
// ExpScale), the sums are formed from memory, a chunk at a time, with exponents no less
// than -1000. That is one instruction in nine for every logit of the others.
template <int THREADS, bool SKIP, int FMT>
RWKV7_DEV void score_row(Chunk<FMT> (&x)[kRowChunks], const void *src, uint32_t n8, float tail, const ExpScale &sc, float M,
                         float own, float &S, float &T, int &n) {
  const float ref = uniform_f(ExpScale::ref(M));
  const bool holds = own == M;  // (wave-uniform)
  S = T = 0.f;
  n = 0;
  auto add = [&](auto most, auto arg, float v, float &s, float &t) {
    const float y = arg(v);
    float e = __builtin_amdgcn_exp2f(y);
    if (decltype(most)::value) {
      const bool is = v == M;
      n += is;
      e = is ? 0.f : e;
    }
    s += e;
    t = fmaf(e, y, t);
  };
  auto chunk = [&](auto most, auto arg, const Chunk<FMT> &c) {
    float f[kRowChunk], s[2] = {0.f, 0.f}, t[2] = {0.f, 0.f};
    c.get(f);
#pragma unroll
    for (int e = 0; e < kRowChunk; ++e) add(most, arg, f[e], s[e & 1], t[e & 1]);
    S += s[0] + s[1];
    T += t[0] + t[1];
  };
  const bool near = sc.near(M), has_tail = threadIdx.x < kRowChunk && !(tail == -kInf);
  auto fast = [&](auto most) {
    auto arg = [&](float v) { return near_arg(sc, v, ref); };
    if (has_tail) add(most, arg, tail, S, T);
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) {
      if (SKIP && c > 0 && c * THREADS >= (int)n8) break;
      Chunk<FMT> y = x[c];
      if (decltype(most)::value) y.opaque();  // (else what both arms unpack alike would go before them, a row's worth)
      if (c * THREADS + (int)threadIdx.x < (int)n8) chunk(most, arg, y);
    }
  };
  if (near) {
    if (holds) fast(BoolConst<true>());
    else fast(BoolConst<false>());
    const float2 st = wave_sum2(S, T);
    S = st.x;
    T = st.y;
  }
  if (!near || (T != T && S == S)) {
    S = T = 0.f;
    n = 0;
    auto arg = [&](float v) { return fmaxf(score_arg(sc, v, ref), v == v ? -1000.f : v); };
    if (has_tail) add(BoolConst<true>(), arg, tail, S, T);
#pragma unroll 1
    for (uint32_t b = threadIdx.x; b < n8; b += THREADS) {
      Chunk<FMT> y;
      y.load_whole(src, b);
      chunk(BoolConst<true>(), arg, y);
    }
    const float2 st = wave_sum2(S, T);
    S = st.x;
    T = st.y;
  }
  n = holds ? (int)wave_sum((float)n) : 0;
}

// The waves joined, by one wave. (A count of 2^24 or less is a float.)
template <int WAVES>
RWKV7_DEV RowSums join_sums(const ScoreLds &s, const ExpScale &sc, float M, int lane) {
  RowSums r;
  const bool in = lane < WAVES;
  r.S = uniform_d(wave_sum_d(in ? (double)s.S[lane] : 0.0));
  r.T = uniform_d(wave_sum_d(in ? (double)s.T[lane] : 0.0));
  r.n = uniform_d(wave_sum_d(in ? (double)s.n[lane] : 0.0));
  r.M = M;
  const float ref = ExpScale::ref(M);
  r.at = (double)score_arg(sc, ref, ref);
  r.slope = kLn2 * sc.more;
  return r;
}

struct RowScore {
  double log_S;  // log sum exp(a (z - M))
  double H;
  bool none;     // every logit is -inf
};

RWKV7_DEV RowScore row_score(const RowSums &r) {
  RowScore o;
  o.none = r.M == -kInf && r.S == 0.0;
  // The exponents' factor is a float, 1.3e-8 less than log2(e): at a mean exponent of -10 a
  // bias of 1e-7 in S, which T makes up for. (H would need a third sum; its two terms are
  // left as they are together, off by that 1.3e-8 times the variance of log q.)
  const double up = exp2_d(-r.at), T1 = up * (r.T - r.at * r.S), more = r.slope * T1;
  const double S1 = fma(r.S, up, more), S = r.n + S1, mean = T1 * rcp_d(S - more);
  // (NaN among the logits makes the sum NaN)
  o.log_S = o.none ? 0.0 : S == S && r.M < kInf ? log_n_plus(r.n, S1) : __builtin_nan("");
  o.H = o.none ? 0.0 : o.log_S - (kLn2 + r.slope) * mean;
  return o;
}

// For the gradient, without a logarithm: the sum of the powers as score_arg() forms them, and
// H less its logarithm, which is the sums' quotient alone. (total is NaN where log_S is.)
struct RowCentre {
  double total, centre;
};
RWKV7_DEV RowCentre row_centre(const RowSums &r) {
  const double one = exp2_frac(r.at), T1 = r.T - r.at * r.S, S = fma(r.n, one, r.S);  // (|at| <= 2^-4)
  return {r.M < kInf ? fma(r.slope, T1, S) : __builtin_nan(""), -(kLn2 + r.slope) * T1 * rcp_d(S) - kLn2 * r.at};
}

// log q of a logit
RWKV7_DEV double log_prob(const RowScore &o, double a, float z, float M) {
  return o.none ? -__builtin_inf() : a * ((double)z - (double)M) - o.log_S;
}

}  // namespace rwkv7
