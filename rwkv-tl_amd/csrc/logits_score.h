// A row's log probabilities and entropy from sums about its largest logit, shared by
// the operators that give them.
//
// With M the largest logit, n logits alike to it and y_j = a (z_j - M) log2(e) <= 0:
//   S = sum 2^y = n + S',  T = sum y 2^y = T'      (S', T': over the others)
//   log q_j = ln 2 (y_j - log2 S),   H = -sum q log q = ln 2 (log2 S - T / S)
// Both terms of H are positive, and S' is summed without the n: a token of
// probability 1 - 1e-9 has log q = -log1p(S') and H to the sums' own rounding (as
// 1 + S' in 32 bits both would be 0). Sums of a wave are in 32 bits, and joined, with
// all that follows, in 64.
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

struct ScoreLds {
  float m[kMaxWaves], S[kMaxWaves], T[kMaxWaves];
  int n[kMaxWaves];
};

// What a wave has of the row beside the largest logits: S' and T' about M as
// ExpScale::with() forms its exponents, which lie `at` (their own value at M) above y.
struct RowSums {
  double S, T, n, at;
  float M;
};

// The exponent of an element, and of M, in 32 bits; F: with()'s far.
template <bool FAR>
RWKV7_DEV float score_arg(const ExpScale &sc, float x, float M, float R) {
  return FAR ? (x - M) * sc.kf : fmaf(x, sc.kf, -R);
}

// Sums of a wave's row about M (wave-uniform, the largest of all waves, `own` this
// wave's largest). A masked element's exponent, -inf, is taken as -1000: 0 times it
// is 0. A NaN among the logits makes S NaN; M is the largest of the others.
template <int THREADS, bool SKIP, int FMT>
RWKV7_DEV void score_row(Chunk<FMT> (&x)[kRowChunks], uint32_t n8, float tail, const ExpScale &sc, float M, float own,
                         float &S, float &T, int &n) {
  S = T = 0.f;
  n = 0;
  const float ref = uniform_f(ExpScale::ref(M));
  auto sums = [&](auto far, auto most) {
    constexpr bool kFar = decltype(far)::value, kMost = decltype(most)::value;
    const float R = ref * sc.kf;
    auto add = [&](float v, float &s, float &t) {
      const float y = score_arg<kFar>(sc, v, ref, R);
      float e = __builtin_amdgcn_exp2f(y);
      if (kMost) {
        const bool is = v == M;
        n += is;
        e = is ? 0.f : e;
      }
      s += e;
      t = fmaf(e, fmaxf(y, -1000.f), t);
    };
    add(tail, S, T);
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) {
      if (SKIP && c > 0 && c * THREADS >= (int)n8) break;
      float f[kRowChunk];
      if (kMost) x[c].opaque();  // (else what both arms unpack alike would go before them, a row's worth)
      x[c].template get<kFar>(f);
      float s[2] = {0.f, 0.f}, t[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < kRowChunk; ++e) add(f[e], s[e & 1], t[e & 1]);
      S += s[0] + s[1];
      T += t[0] + t[1];
    }
  };
  const bool holds = own == M, near = sc.near(M);  // (wave-uniform)
  if (near) {
    if (holds) sums(BoolConst<false>(), BoolConst<true>());
    else sums(BoolConst<false>(), BoolConst<false>());
  } else {
    if (holds) sums(BoolConst<true>(), BoolConst<true>());
    else sums(BoolConst<true>(), BoolConst<false>());
  }
  const float2 st = wave_sum2(S, T);
  S = st.x;
  T = st.y;
  if (holds) n = (int)wave_sum((float)n);
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
  r.at = sc.near(M) ? (double)score_arg<false>(sc, ref, ref, ref * sc.kf) : 0.0;
  return r;
}

struct RowScore {
  double log_S;  // log sum exp(a (z - M))
  double H;
  double total;  // sum of the exponents' powers as score_arg forms them, and its logarithm
  double log_total;
  bool none;     // every logit is -inf
};

RWKV7_DEV RowScore row_score(const RowSums &r) {
  RowScore o;
  o.none = r.M == -kInf && r.S == 0.0;
  const double up = exp2_d(-r.at), S1 = r.S * up, T1 = up * (r.T - r.at * r.S), S = r.n + S1;
  // (NaN among the logits makes the sum NaN)
  o.log_S = S == S && r.M < kInf ? log_n_plus(r.n, S1) : __builtin_nan("");
  o.H = o.none ? 0.0 : o.log_S - kLn2 * T1 * rcp_d(S);
  o.total = S * exp2_d(r.at);
  o.log_total = o.log_S + kLn2 * r.at;
  return o;
}

// log q of a logit
RWKV7_DEV double log_prob(const RowScore &o, double a, float z, float M) {
  return o.none ? -__builtin_inf() : a * ((double)z - (double)M) - o.log_S;
}

}  // namespace rwkv7
