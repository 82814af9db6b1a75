// Log probabilities of given tokens, the rows' entropies, and the gradient of both,
// one workgroup per row (with alternatives: top_logits.hip).
//
//   q_j = exp(a z_j - L), L = log sum exp(a z), a = 1 / temperature
//   l = a z_x - L,  H = -sum q log q
//   d (s l + h H) / d z_j = a (s (1 where j = x) - q_j (s + h (log q_j + H)))
// x outside 0 .. V-1: a padded row, l = H = 0 and gradient 0 whatever its logits hold. A
// row of -inf alone: l = -inf, H = 0, gradient 0. NaN or +inf elsewhere: NaN, as in a
// log-softmax.
//
// The row stays in registers: the largest, then the sums about it (logits_score.h), then
// the gradient, with one read and one write of memory. The token's own gradient is
// formed in 64 bits (1 - q of a likely token is what is left of a difference) and
// stored over the row's after a barrier.
//
// Bytes bound it. Measured (kernel trace, us; a large copy moves 5.09 TB/s here): 2039 x 65536 bf16 48
// (5.6 TB/s), with a masked end 96 and with all but 300 masked 105 (-inf: the sums once more, from
// memory), 2000 x 65536 f32 108 (4.9, one workgroup on a CU); with the gradient 4096 x 65536
// bf16 201 and f16 199 (5.4), masked alike 303 and 320, 2000 x 65536 f32 231 (4.5), with that of the entropy 2048 x 65536 bf16
// 102; one row 6.6 and 10.8, 331 x 20011 f32 9.1 and 14.3, chains of load, maximum, sum and
// join. With the logarithms and the token's own gradient before the row's, where a wave
// that holds the row has no registers for them, 4096 x 65536 bf16 took 228-245.
#include "logits_score.h"
#include "rwkv7_kernels.h"

namespace rwkv7 {
namespace {

struct TokenArgs {
  const void *logits;
  int64_t ld;
  int V;
  ExpScale sc;
  double a;
  const int64_t *tokens;
  float *logp, *entropy;  // null: not wanted
  // gradient only: the rows' upstream gradients, null: the same for all
  const float *scale, *entropy_scale;
  float scale0, entropy_scale0;
  void *grad;
  int64_t row0;
};

template <int FMT, int THREADS>
RWKV7_DEV void zero_grad(char *dst, int V) {
  const float zero[kRowChunk] = {};
#pragma unroll 1
  for (uint32_t b = threadIdx.x; b < (uint32_t)V / kRowChunk; b += THREADS) store_chunk<FMT>(dst, b, zero);
  if (threadIdx.x < V % kRowChunk) store_logit<FMT>(dst, V / kRowChunk * kRowChunk + threadIdx.x, 0.f);
}

struct TokenLds {
  ScoreLds s;
  float base, slope;  // the gradient is 2^y (base + slope y), with log q = ln 2 y - log total
};

template <int FMT, int THREADS, bool GRAD>
__global__ __launch_bounds__(THREADS, FMT == 1 ? 4 : 8) void token_kernel(TokenArgs g) {
  __shared__ TokenLds s;
  constexpr int kWaves = THREADS / kWave;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, V = g.V;
  const uint32_t n8 = (uint32_t)V / kRowChunk;
  const int64_t row = g.row0 + blockIdx.x;
  const char *src = static_cast<const char *>(g.logits) + row * g.ld * kLogitBytes<FMT>;
  char *dst = GRAD ? static_cast<char *>(g.grad) + row * (int64_t)V * kLogitBytes<FMT> : nullptr;
  const int64_t id = g.tokens[row];
  float up = 0.f, up_h = 0.f;
  if (GRAD) {
    up = g.scale ? g.scale[row] : g.scale0;
    up_h = g.entropy_scale ? g.entropy_scale[row] : g.entropy_scale0;
  }
  if (id < 0 || id >= V) {  // (block-uniform)
    if (t == 0 && g.logp) g.logp[row] = 0.f;
    if (t == 0 && g.entropy) g.entropy[row] = 0.f;
    if (GRAD) zero_grad<FMT, THREADS>(dst, V);
    return;
  }
  if (GRAD && !g.logp && !g.entropy && up == 0.f && up_h == 0.f) {
    zero_grad<FMT, THREADS>(dst, V);
    return;
  }

  Chunk<FMT> x[kRowChunks];
  load_row<THREADS>(x, src, n8);
  const int tail = t < V % kRowChunk ? (int)n8 * kRowChunk + t : -1;  // this thread's logit behind the eights
  const float xt = tail >= 0 ? load_logit<FMT>(src, tail) : -kInf;
  const float zx = load_logit<FMT>(src, id);

  auto largest = [&](auto most) {
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) {
      if (!GRAD && c > 0 && c * THREADS >= (int)n8) break;
      most.add(x[c]);
    }
    opaque_row(x);
    return most;
  };
  float own;
  if constexpr (GRAD) {  // (bound by its bytes, and short of registers)
    own = wave_max(fmaxf(largest(RowMax<FMT>()).value(), xt));
  } else {
    const PairMax<FMT> pairs = largest(PairMax<FMT>());
    own = wave_max(fmaxf(pairs.value(), xt));
    if (__ballot(!pairs.clean())) own = wave_max(fmaxf(largest(RowMax<FMT>()).value(), xt));
  }
  if (lane == 0) s.s.m[wv] = own;
  __syncthreads();
  const float M = uniform_f(wave_max(lane < kWaves ? s.s.m[lane] : -kInf));

  float S, T;
  int n;
  score_row<THREADS, !GRAD>(x, src, n8, xt, g.sc, M, own, S, T, n);
  if (lane == 0) s.s.S[wv] = S, s.s.T[wv] = T, s.s.n[wv] = n;
  if (GRAD) opaque_row(x);
  __syncthreads();

  // What the row's gradient needs of the sums, by one wave that the others wait for (no
  // more than that: beside the row there are no registers for it, and a spilled one is a
  // trip to memory); all else when the row is stored.
  if (GRAD && wv == 0) {
    const RowSums r = join_sums<kWaves>(s.s, g.sc, M, lane);
    const bool zero = (up == 0.f && up_h == 0.f) || (M == -kInf && r.S == 0.0);
    // log q = ln 2 y - log total
    const RowCentre o = row_centre(r);
    const double f = -g.a * rcp_d(o.total), base = f * ((double)up + (double)up_h * o.centre), slope = f * kLn2 * (double)up_h;
    if (lane == 0) s.base = zero ? 0.f : (float)base, s.slope = zero ? 0.f : (float)slope;
  }
  if (GRAD) __syncthreads();
  auto outputs = [&]() {  // by one wave
    const RowScore r = row_score(join_sums<kWaves>(s.s, g.sc, M, lane));
    const double lp = log_prob(r, g.a, zx, M);
    if (lane == 0 && g.logp) g.logp[row] = (float)lp;
    if (lane == 0 && g.entropy) g.entropy[row] = (float)r.H;
    if (GRAD && !(r.none || (up == 0.f && up_h == 0.f))) {
      double grad = g.a * (double)up * one_minus_exp(lp);
      if (up_h != 0.f && lp != -__builtin_inf())  // (NaN stays NaN)
        grad -= g.a * (double)up_h * (lp == lp ? exp2_d(1.4426950408889634 * lp) : lp) * (lp + r.H);
      if (lane == 0) store_logit<FMT>(dst, id, (float)grad);
    }
  };
  if (!GRAD) {
    if (wv == 0) outputs();
    return;
  }
  const float base = uniform_f(s.base), slope = uniform_f(s.slope);
  if (base == 0.f && slope == 0.f) {  // a row that counts for nothing: zeros, not 0 * NaN
    zero_grad<FMT, THREADS>(dst, V);
  } else {
    const float ref = uniform_f(ExpScale::ref(M));
    // (an exponent of -inf, a masked logit's, is taken as -1000: 0 times it is 0)
    auto sloped = [&](float y) { return __builtin_amdgcn_exp2f(y) * fmaf(slope, fmaxf(y, -1000.f), base); };
    auto put = [&](auto flat) {
      constexpr bool kFlat = decltype(flat)::value;
      auto one = [&](float v) {
        const float y = near_arg(g.sc, v, ref);
        return kFlat ? __builtin_amdgcn_exp2f(y) * base : sloped(y);
      };
#pragma unroll
      for (int c = 0; c < kRowChunks; ++c) {
        if (c > 0 && c * THREADS >= (int)n8) break;
        float f[kRowChunk];
        if (!kFlat) x[c].opaque();
        x[c].get(f);
#pragma unroll
        for (int e = 0; e < kRowChunk; ++e) f[e] = one(f[e]);
        const uint32_t b = c * THREADS + t;
        if ((c + 1) * THREADS <= (int)n8) store_chunk<FMT>(dst, b, f);
        else if (b < n8) store_chunk<FMT>(dst, b, f);
      }
    };
    if (g.sc.near(M)) {
      if (slope == 0.f) put(BoolConst<true>());
      else put(BoolConst<false>());
    } else {  // far from 0, from memory
#pragma unroll 1
      for (uint32_t b = t; b < n8; b += THREADS) {
        Chunk<FMT> y;
        float f[kRowChunk];
        y.load_whole(src, b);
        y.get(f);
#pragma unroll
        for (int e = 0; e < kRowChunk; ++e) f[e] = sloped(score_arg(g.sc, f[e], ref));
        store_chunk<FMT>(dst, b, f);
      }
    }
    if (tail >= 0) store_logit<FMT>(dst, tail, sloped(score_arg(g.sc, xt, ref)));
  }
  __syncthreads();  // the row's own stores come before the token's
  if (wv == 0) outputs();
}

template <int FMT, int THREADS>
void launch_t(const TokenArgs &g, int N, hipStream_t st) {
  if (g.grad) token_kernel<FMT, THREADS, true><<<N, THREADS, 0, st>>>(g);
  else token_kernel<FMT, THREADS, false><<<N, THREADS, 0, st>>>(g);
}

template <int FMT>
void launch_f(const TokenArgs &g, int N, hipStream_t st) {
  switch (row_threads(g.V)) {
    case 256: launch_t<FMT, 256>(g, N, st); break;
    case 512: launch_t<FMT, 512>(g, N, st); break;
    default: launch_t<FMT, 1024>(g, N, st); break;
  }
}

int launch_rows(TokenArgs g, int dtype, int N, hipStream_t st) {
  for (; g.row0 < N; g.row0 += kLaunchRows) {
    const int n = N - g.row0 < kLaunchRows ? (int)(N - g.row0) : kLaunchRows;
    switch (dtype) {
      case 0: launch_f<0>(g, n, st); break;
      case 1: launch_f<1>(g, n, st); break;
      default: launch_f<2>(g, n, st); break;
    }
    RWKV7_CHECK_LAUNCH();
  }
  return RWKV7_OK;
}

}  // namespace
}  // namespace rwkv7

extern "C" int rwkv7_token_logprobs(const void *logits, int32_t logits_dtype, int64_t ld, int32_t N, int32_t V,
                                    const int64_t *tokens, double temperature, int32_t k, float *logp, float *entropy,
                                    float *top_logp, int64_t *top_idx, void *stream) {
  using namespace rwkv7;
  if (!logits || !tokens || !logp || !entropy || logits_dtype < 0 || logits_dtype > 2) return RWKV7_EINVAL;
  if (!(temperature >= 1e-30 && temperature <= 1e30)) return RWKV7_EINVAL;
  if (N < 1 || V < 1 || V > kRowMaxV || ld < V || k < 0) return RWKV7_ESHAPE;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (k > 0) {
    if (!top_logp || !top_idx) return RWKV7_EINVAL;
    return launch_top_scores(logits, logits_dtype, ld, N, V, tokens, temperature, k, logp, entropy, top_logp, top_idx, st);
  }
  const double a = 1.0 / temperature;
  return launch_rows({logits, ld, V, ExpScale::of(a), a, tokens, logp, entropy}, logits_dtype, N, st);
}

extern "C" int rwkv7_token_logprobs_grad(const void *logits, int32_t logits_dtype, int64_t ld, int32_t N, int32_t V,
                                         const int64_t *tokens, double temperature, const float *scale, float scale0,
                                         const float *entropy_scale, float entropy_scale0, float *logp, float *entropy,
                                         void *grad, void *stream) {
  using namespace rwkv7;
  if (!logits || !tokens || !grad || logits_dtype < 0 || logits_dtype > 2) return RWKV7_EINVAL;
  if (!(temperature >= 1e-30 && temperature <= 1e30)) return RWKV7_EINVAL;
  if (N < 1 || V < 1 || V > kRowMaxV || ld < V) return RWKV7_ESHAPE;
  const double a = 1.0 / temperature;
  return launch_rows({logits, ld, V, ExpScale::of(a), a, tokens, logp, entropy, scale, entropy_scale, scale0, entropy_scale0, grad},
                     logits_dtype, N, static_cast<hipStream_t>(stream));
}
