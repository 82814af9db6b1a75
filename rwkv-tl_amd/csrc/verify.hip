// Verification of drafted tokens against a target model's probabilities, from
// given random numbers (speculative sampling).
//
// For sequence b with len drafted tokens x_0 .. x_{len-1}: p_i = softmax of the
// target's logits after i of them over temperature T, q_i = softmax of the draft
// model's over its own, or one-hot at x_i where it drafted without a draw. x_i
// is accepted while u_i q_i(x_i) < p_i(x_i). The token after the accepted ones
// is drawn from max(p_j - q_j, 0) at the first rejected j (from p_j if that is 0
// everywhere), from p_len if all are accepted: the first v whose inclusive sum
// exceeds u_K times the whole. The tokens then follow p exactly. T <= 0: x_i is
// accepted while it is the target's argmax (lowest id of a tie), and the next
// token is the argmax.
//
// The sums and the draw are in 64 bits: among 65536 tokens the borders of the
// cumulative sum lie within 1e-9 of each other in the tail, where f32 sums (1e-7)
// would draw another token than the one that u stands for. One 64-bit fma costs
// as much as one 32-bit fma on this machine, so an exponential of ~18 of them
// takes about as long as reading its logit.
//
// NaN counts as -inf (never drawn, never accepted). A drafted id outside the
// vocabulary is rejected, a row without a finite logit has no probability: its
// drafted token is rejected, and the next token falls to 0 if nothing is left to
// draw from.
//
// verify_stats_kernel: a slice of a row per workgroup: its largest logit and the
//   sum of the exponentials about it (greedy: largest logit and its first id).
// verify_rest_kernel: a slice of each sequence's decisive row: every workgroup
//   joins the sums of its sequence's rows and decides how many tokens are
//   accepted; the slice's sum of max(p - q, 0).
// verify_draw_kernel: one workgroup per sequence: decides again, finds the slice
//   in which the sum crosses, and in it the token.
#include "logits_rows.h"
#include "rwkv7_kernels.h"

namespace rwkv7 {
namespace {

constexpr int kVerThreads = 256;
constexpr int kVerChunks = 4;
constexpr int kVerE = kVerChunks * kRowChunk;       // logits per thread of a slice
constexpr int kSlice = kVerThreads * kVerE;         // 8192
constexpr int kMaxSlices = kRowMaxV / kSlice;       // 8
constexpr int kVerMaxK = kWave - 1;                 // a lane per drafted token and one for the row behind them

struct VerifyArgs {
  const void *target, *draft;  // draft null: one-hot
  int64_t tb, tr, db, dr;      // strides of a sequence and of a row, in elements
  const int64_t *tok;
  const float *u;
  const int64_t *len;          // null: K
  int B, K, V, G;              // G slices of a row
  double kt, kd;               // log2(e) / temperature of target and draft; kt <= 0: greedy
  int64_t *out, *accepted;
  // workspace
  float *m;                    // [rows][G] largest logit; rows: B (K + 1) of the target, B K of the draft
  double *sum;                 // [rows][G] sum of exponentials about m (greedy: first id of the largest)
  double *rest;                // [B][G] sums of max(p - q, 0)
};

// 2^(k (x - m)): 1 at the largest logit (also +inf), 0 for -inf and NaN.
RWKV7_DEV double weight(float x, float m, double k) {
  return x == m ? (m > -kInf ? 1.0 : 0.0) : exp2_d(((double)x - (double)m) * k);
}

// Joined sums of the slices of one row.
struct RowSum {
  float m;
  double S;
};
RWKV7_DEV RowSum join_row(const VerifyArgs &a, int64_t r, double k) {
  RowSum j = {-kInf, 0.0};
  for (int s = 0; s < a.G; ++s) j.m = fmaxf(j.m, a.m[r * a.G + s]);
  for (int s = 0; s < a.G; ++s) {
    const float ms = a.m[r * a.G + s];
    j.S += a.sum[r * a.G + s] * weight(ms, j.m, k);
  }
  return j;
}

RWKV7_DEV int drafted(const VerifyArgs &a, int b) {
  if (!a.len) return a.K;
  const int64_t n = a.len[b];
  return n < 0 ? 0 : n > a.K ? a.K : (int)n;
}

template <int FMT>
RWKV7_DEV const void *target_row(const VerifyArgs &a, int b, int i) {
  return static_cast<const char *>(a.target) + (b * a.tb + i * a.tr) * kLogitBytes<FMT>;
}
template <int FMT>
RWKV7_DEV const void *draft_row(const VerifyArgs &a, int b, int i) {
  return static_cast<const char *>(a.draft) + (b * a.db + i * a.dr) * kLogitBytes<FMT>;
}

template <int FMT, bool GREEDY>
__global__ __launch_bounds__(kVerThreads) void verify_stats_kernel(VerifyArgs a) {
  __shared__ float s_m[kVerThreads / kWave];
  __shared__ double s_sum[kVerThreads / kWave];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, V = a.V, g = blockIdx.x;
  const int64_t r = blockIdx.y;
  const int64_t nt = (int64_t)a.B * (a.K + 1);
  const bool tgt = r < nt;
  const int per = tgt ? a.K + 1 : a.K;
  const int b = (int)((tgt ? r : r - nt) / per), i = (int)((tgt ? r : r - nt) % per);
  const int len = drafted(a, b);
  if (i >= (tgt ? len + 1 : len)) return;  // a row that no decision looks at
  const void *row = tgt ? target_row<FMT>(a, b, i) : draft_row<FMT>(a, b, i);
  const uint32_t n8 = (uint32_t)V / kRowChunk;
  Chunk<FMT> x[kVerChunks];
#pragma unroll
  for (int c = 0; c < kVerChunks; ++c) x[c].load(row, (g * kVerChunks + c) * kVerThreads + t, n8);
  const int tail = g == a.G - 1 && t < V % kRowChunk ? (int)n8 * kRowChunk + t : -1;
  const float xt = tail >= 0 ? load_logit<FMT>(row, tail) : -kInf;
  float m = fmaxf(xt, -kInf);
#pragma unroll
  for (int c = 0; c < kVerChunks; ++c) {
    float f[kRowChunk];
    x[c].get(f);
#pragma unroll
    for (int e = 0; e < kRowChunk; ++e) m = fmaxf(m, f[e]);
  }
  m = wave_max(m);
  if (lane == 0) s_m[wv] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kVerThreads / kWave; ++w) m = fmaxf(m, s_m[w]);
  double sum = 0.0;
  if (GREEDY) {
    int at = V;  // first id of the largest
#pragma unroll
    for (int c = kVerChunks - 1; c >= 0; --c) {
      float f[kRowChunk];
      x[c].get(f);
#pragma unroll
      for (int e = kRowChunk - 1; e >= 0; --e)
        if (f[e] == m) at = (int)((g * kVerChunks + c) * kVerThreads + t) * kRowChunk + e;
    }
    if (at == V && tail >= 0 && xt == m) at = tail;
    if (m == -kInf) at = V;  // nothing but -inf and NaN
    sum = -wave_max_d(-(double)at);
  } else {
    const double k = tgt ? a.kt : a.kd;
    sum = tail >= 0 ? weight(xt, m, k) : 0.0;
#pragma unroll
    for (int c = 0; c < kVerChunks; ++c) {
      float f[kRowChunk];
      x[c].get(f);
#pragma unroll
      for (int e = 0; e < kRowChunk; ++e) sum += weight(f[e], m, k);
    }
    sum = wave_sum_d(sum);
  }
  if (lane == 0) s_sum[wv] = sum;
  __syncthreads();
  if (t == 0) {
#pragma unroll
    for (int w = 1; w < kVerThreads / kWave; ++w) sum = GREEDY ? fmin(sum, s_sum[w]) : sum + s_sum[w];
    a.m[r * a.G + g] = m;
    a.sum[r * a.G + g] = sum;
  }
}

// What wave 0 finds out about sequence b: the accepted tokens, and about the row
// behind them.
struct Decision {
  int n, rejected;      // accepted tokens; whether the next was drafted and rejected
  float mp, mq;
  double ip, iq;        // 1 / sum of the row's exponentials, 0 for an empty row; iq 0 without a draft row
  int x;                // the rejected token of a one-hot draft, else -1
};

template <int FMT>
RWKV7_DEV void decide(const VerifyArgs &a, int b, Decision *d) {
  const int lane = threadIdx.x;
  if (lane >= kWave) return;
  const int len = drafted(a, b);
  RowSum p = {-kInf, 0.0}, q = {-kInf, 0.0};
  bool ok = false;
  if (lane <= len) p = join_row(a, (int64_t)b * (a.K + 1) + lane, a.kt);
  if (lane < len) {
    const int64_t x = a.tok[(int64_t)b * a.K + lane];
    const bool in = x >= 0 && x < a.V;
    const double px = in && p.S > 0.0 ? weight(load_logit<FMT>(target_row<FMT>(a, b, lane), x), p.m, a.kt) / p.S : 0.0;
    double qx = 1.0;
    if (a.draft) {
      q = join_row(a, (int64_t)a.B * (a.K + 1) + (int64_t)b * a.K + lane, a.kd);
      qx = in && q.S > 0.0 ? weight(load_logit<FMT>(draft_row<FMT>(a, b, lane), x), q.m, a.kd) / q.S : 0.0;
    }
    ok = px > 0.0 && (double)a.u[(int64_t)b * (a.K + 1) + lane] * qx < px;
  }
  const u64 bad = ~__ballot(ok);  // (lane len is never ok)
  const int n = __ffsll(bad) - 1;
  if (lane == n) {
    d->n = n;
    d->rejected = n < len;
    d->mp = p.m, d->mq = q.m;
    d->ip = p.S > 0.0 ? 1.0 / p.S : 0.0;
    d->iq = q.S > 0.0 ? 1.0 / q.S : 0.0;
    d->x = -1;
    if (n < len && !a.draft) {
      const int64_t x = a.tok[(int64_t)b * a.K + n];
      if (x >= 0 && x < a.V) d->x = (int)x;
    }
  }
}

// max(p - q, 0) of one logit; id: its index.
RWKV7_DEV double residual(const VerifyArgs &a, const Decision &d, float xp, float xq, int id) {
  double r = weight(xp, d.mp, a.kt) * d.ip;
  if (a.draft) r = fmax(r - weight(xq, d.mq, a.kd) * d.iq, 0.0);
  return id == d.x ? 0.0 : r;
}

template <int FMT>
__global__ __launch_bounds__(kVerThreads) void verify_rest_kernel(VerifyArgs a) {
  __shared__ Decision s_d;
  __shared__ double s_sum[kVerThreads / kWave];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, V = a.V, g = blockIdx.x, b = blockIdx.y;
  decide<FMT>(a, b, &s_d);
  __syncthreads();
  const Decision d = s_d;
  if (!d.rejected) return;
  const void *pr = target_row<FMT>(a, b, d.n), *qr = a.draft ? draft_row<FMT>(a, b, d.n) : pr;
  const uint32_t n8 = (uint32_t)V / kRowChunk;
  double sum = 0.0;
#pragma unroll 1
  for (int c = 0; c < kVerChunks; ++c) {
    const uint32_t e8 = (g * kVerChunks + c) * kVerThreads + t;
    if (e8 >= n8) break;
    Chunk<FMT> xp, xq;
    xp.load(pr, e8, n8);
    xq.load(qr, e8, n8);
    float fp[kRowChunk], fq[kRowChunk];
    xp.get(fp);
    xq.get(fq);
#pragma unroll
    for (int e = 0; e < kRowChunk; ++e) sum += residual(a, d, fp[e], fq[e], (int)e8 * kRowChunk + e);
  }
  if (g == a.G - 1 && t < V % kRowChunk) {
    const int id = (int)n8 * kRowChunk + t;
    sum += residual(a, d, load_logit<FMT>(pr, id), load_logit<FMT>(qr, id), id);
  }
  sum = wave_sum_d(sum);
  if (lane == 0) s_sum[wv] = sum;
  __syncthreads();
  if (t == 0) {
#pragma unroll
    for (int w = 1; w < kVerThreads / kWave; ++w) sum += s_sum[w];
    a.rest[(int64_t)b * a.G + g] = sum;
  }
}

template <int FMT>
__global__ __launch_bounds__(kVerThreads) void verify_draw_kernel(VerifyArgs a) {
  __shared__ Decision s_d;
  __shared__ double s_slice[kMaxSlices + 1], s_wave[kVerThreads / kWave];
  __shared__ int s_first, s_last;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, V = a.V, b = blockIdx.x;
  decide<FMT>(a, b, &s_d);
  __syncthreads();
  const Decision d = s_d;
  const int64_t r = (int64_t)b * (a.K + 1) + d.n;
  // the slices' sums of what is drawn from: p - q, or p itself
  bool from_p = !d.rejected;
  if (t < a.G && d.rejected) s_slice[t] = a.rest[(int64_t)b * a.G + t];
  __syncthreads();
  if (d.rejected) {
    double all = 0.0;
    for (int s = 0; s < a.G; ++s) all += s_slice[s];
    from_p = !(all > 0.0);
    __syncthreads();
  }
  if (from_p && t < a.G) s_slice[t] = a.sum[r * a.G + t] * weight(a.m[r * a.G + t], d.mp, a.kt) * d.ip;
  if (t == 0) s_first = V, s_last = -1;
  __syncthreads();
  double all = 0.0;
  for (int s = 0; s < a.G; ++s) all += s_slice[s];
  const double goal = (double)a.u[(int64_t)b * (a.K + 1) + a.K] * all;
  // the first slice in which the inclusive sum exceeds the goal; none (u >= 1, or
  // rounding): the last one with any weight
  int g = -1, with = 0;
  double before = 0.0, base = 0.0;
  for (int s = 0; s < a.G; ++s) {
    if (s_slice[s] > 0.0) with = s;
    if (g < 0 && before + s_slice[s] > goal) g = s, base = before;
    before += s_slice[s];
  }
  const bool none = g < 0;
  if (none) g = with;
  // its logits, 32 consecutive ones a thread (and the row's last few)
  const void *pr = target_row<FMT>(a, b, d.n), *qr = a.draft && d.rejected ? draft_row<FMT>(a, b, d.n) : pr;
  const int i0 = g * kSlice + t * kVerE;
  auto at = [&](int id) {
    const float xp = load_logit<FMT>(pr, id);
    return from_p ? weight(xp, d.mp, a.kt) * d.ip : residual(a, d, xp, load_logit<FMT>(qr, id), id);
  };
  double own = 0.0;
  int last = -1;
#pragma unroll 4
  for (int e = 0; e < kVerE; ++e) {
    const int id = i0 + e;
    if (id >= V) break;
    const double w = at(id);
    own += w;
    if (w > 0.0) last = id;
  }
  // inclusive sums over the threads
  double inc = own;
#pragma unroll
  for (int s = 1; s < kWave; s <<= 1) {
    const u64 v = __builtin_bit_cast(u64, inc);
    const int lo = __shfl_up((int)(uint32_t)v, s), hi = __shfl_up((int)(uint32_t)(v >> 32), s);
    if (lane >= s) inc += __builtin_bit_cast(double, (u64)(uint32_t)lo | ((u64)(uint32_t)hi << 32));
  }
  if (lane == kWave - 1) s_wave[wv] = inc;
  __syncthreads();
  for (int w = 0; w < wv; ++w) base += s_wave[w];
  if (last >= 0) atomicMax(&s_last, last);
  if (!none && own > 0.0 && base + inc > goal) {
    double acc = base + (inc - own);
    int found = last;  // (by rounding, the running sum may end just below the goal)
    for (int e = 0; e < kVerE && i0 + e < V; ++e) {
      const double w = at(i0 + e);
      acc += w;
      if (w > 0.0 && acc > goal) {
        found = i0 + e;
        break;
      }
    }
    atomicMin(&s_first, found);
  }
  __syncthreads();
  const int next = s_first < V ? s_first : s_last >= 0 ? s_last : 0;
  if (t <= a.K) a.out[(int64_t)b * (a.K + 1) + t] = t < d.n ? a.tok[(int64_t)b * a.K + t] : t == d.n ? next : -1;
  if (t == 0) a.accepted[b] = d.n;
}

// Greedy: one wave per sequence, a lane per drafted token.
__global__ __launch_bounds__(kWave) void verify_greedy_kernel(VerifyArgs a) {
  const int lane = threadIdx.x, b = blockIdx.x, len = drafted(a, b);
  int best = a.V;
  if (lane <= len) {
    const int64_t r = (int64_t)b * (a.K + 1) + lane;
    float m = -kInf;
    for (int s = 0; s < a.G; ++s) {
      const float v = a.m[r * a.G + s];
      if (v > m) m = v, best = (int)a.sum[r * a.G + s];
    }
    if (best >= a.V) best = 0;
  }
  const int64_t x = lane < a.K ? a.tok[(int64_t)b * a.K + lane] : -1;
  const bool ok = lane < len && x == best;
  const int n = __ffsll(~__ballot(ok)) - 1;
  if (lane <= a.K) a.out[(int64_t)b * (a.K + 1) + lane] = lane < n ? x : lane == n ? best : -1;
  if (lane == 0) a.accepted[b] = n;
}

int slices(int V) { return (V + kSlice - 1) / kSlice; }

template <int FMT>
int launch_verify(const VerifyArgs &a, hipStream_t st) {
  const int64_t rows = (int64_t)a.B * (a.K + 1) + (a.draft ? (int64_t)a.B * a.K : 0);
  const dim3 grid(a.G, (unsigned)rows);
  if (a.kt <= 0.0) {
    verify_stats_kernel<FMT, true><<<grid, kVerThreads, 0, st>>>(a);
    RWKV7_CHECK_LAUNCH();
    verify_greedy_kernel<<<a.B, kWave, 0, st>>>(a);
    RWKV7_CHECK_LAUNCH();
    return RWKV7_OK;
  }
  verify_stats_kernel<FMT, false><<<grid, kVerThreads, 0, st>>>(a);
  RWKV7_CHECK_LAUNCH();
  if (a.K > 0) {
    verify_rest_kernel<FMT><<<dim3(a.G, a.B), kVerThreads, 0, st>>>(a);
    RWKV7_CHECK_LAUNCH();
  }
  verify_draw_kernel<FMT><<<a.B, kVerThreads, 0, st>>>(a);
  RWKV7_CHECK_LAUNCH();
  return RWKV7_OK;
}

int64_t al256(int64_t x) { return (x + 255) / 256 * 256; }

}  // namespace
}  // namespace rwkv7

extern "C" int64_t rwkv7_verify_workspace_bytes(int32_t B, int32_t K, int32_t V) {
  using namespace rwkv7;
  if (B < 1 || K < 0 || K > kVerMaxK || V < 1 || V > kRowMaxV) return 0;
  const int64_t rg = (int64_t)B * (2 * K + 1) * slices(V);
  return al256(rg * 4) + al256(rg * 8) + al256((int64_t)B * slices(V) * 8);
}

extern "C" int rwkv7_verify(const void *target, int64_t target_b, int64_t target_r, const void *draft, int64_t draft_b,
                            int64_t draft_r, int32_t logits_dtype, const int64_t *tokens, const float *uniforms,
                            const int64_t *lengths, int32_t B, int32_t K, int32_t V, double temperature,
                            double draft_temperature, int64_t *out, int64_t *accepted, void *workspace,
                            int64_t workspace_bytes, void *stream) {
  using namespace rwkv7;
  if (!target || !out || !accepted || !workspace || logits_dtype < 0 || logits_dtype > 2) return RWKV7_EINVAL;
  if (temperature != temperature || draft_temperature != draft_temperature) return RWKV7_EINVAL;
  const bool greedy = !(temperature > 0.0);
  if ((K > 0 && !tokens) || (!greedy && !uniforms)) return RWKV7_EINVAL;
  const bool soft = !greedy && draft && K > 0 && draft_temperature > 0.0;  // a draft that was drawn
  if (!greedy && (temperature < 1e-30 || temperature > 1e30)) return RWKV7_EINVAL;
  if (soft && (draft_temperature < 1e-30 || draft_temperature > 1e30)) return RWKV7_EINVAL;
  if (B < 1 || K < 0 || K > kVerMaxK || V < 1 || V > kRowMaxV || (int64_t)B * (2 * K + 1) > 65535) return RWKV7_ESHAPE;
  if (target_r < V || target_b < 0 || (soft && (draft_r < V || draft_b < 0))) return RWKV7_ESHAPE;
  if (workspace_bytes < rwkv7_verify_workspace_bytes(B, K, V)) return RWKV7_EWORKSPACE;
  constexpr double kLog2E = 1.4426950408889634;
  const int G = slices(V);
  const int64_t rg = (int64_t)B * (2 * K + 1) * G;
  char *w = static_cast<char *>(workspace);
  VerifyArgs a;
  a.target = target, a.draft = soft ? draft : nullptr;
  a.tb = target_b, a.tr = target_r, a.db = draft_b, a.dr = draft_r;
  a.tok = tokens, a.u = uniforms, a.len = lengths;
  a.B = B, a.K = K, a.V = V, a.G = G;
  a.kt = greedy ? 0.0 : kLog2E / temperature;
  a.kd = soft ? kLog2E / draft_temperature : 0.0;
  a.out = out, a.accepted = accepted;
  a.m = reinterpret_cast<float *>(w);
  a.sum = reinterpret_cast<double *>(w + al256(rg * 4));
  a.rest = reinterpret_cast<double *>(w + al256(rg * 4) + al256(rg * 8));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (logits_dtype) {
    case 0: return launch_verify<0>(a, st);
    case 1: return launch_verify<1>(a, st);
    default: return launch_verify<2>(a, st);
  }
}
