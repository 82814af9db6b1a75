// Distillation from a teacher's top logits: the divergence of a student's
// distribution from them, and its gradient, one workgroup per row.
//
// Student: q_j = exp(a z_j - L), L = log sum_j exp(a z_j), a = 1 / temperature.
// Teacher: entries k < K of ids i_k and logits t_k; one whose id is outside
// 0 .. V-1 is absent. I is the set of ids present.
//   lse given (Lt, over the teacher's whole vocabulary): p_k = exp(a t_k - Lt),
//     P = sum p_k, and R = 1 - P is the teacher's mass outside I (0 below
//     least_rest, which an f32 Lt cannot tell from none, and 0 where I is the whole
//     vocabulary), held against the student's own mass there, 1 - Q = sum_{j not
//     in I} q_j.
//   no lse: p = softmax of a t over the present entries; P = 1, R = 0.
//   loss = sum_k p_k (log p_k - log q_{i_k}) + R (log R - log(1 - Q))
//   d loss / d z_j = a ((P + R) q_j - sum_{k: i_k = j} p_k)      j in I
//                  = a q_j (P + R - R / (1 - Q))                  else
// A row without a present entry or without mass (no lse and entries of -inf alone, or an
// lse of kNoTeacher or less: a teacher's row that a mask leaves nothing of) has loss 0
// and gradient 0, whatever its logits hold. NaN elsewhere makes its row NaN, as in a
// log-softmax.
//
// 1 - Q is never formed as a difference: the row's elements in I are taken out
// (each thread has a word in LDS that marks them) before the sum, and I enters
// through the entries. The row stays in registers between the sum and the
// gradient, so a pass reads the logits once and writes the gradient once; the
// entries' own gradients are stored over it after a barrier.
//
// The row's exponentials are in 32 bits, and so are the sums of a wave; waves are
// joined, and the entries' exponentials, products and gradients formed, in 64: a
// listed id's gradient is what is left of q - p, and the loss what is left of terms
// of both signs (in 32 bits a loss of 331 x 20011 f32 was off by 3.5e-6 of itself,
// now by 1.2e-7).
//
// Measured (kernel trace, us; a large copy moves 5.05 TB/s here): loss and gradient of
// 4096 x 65536 bf16 216, 5.0 TB/s: the bytes (vector units busy 64 %). Loss of 1021 x
// 65536 f16 29.8, 4.5 TB/s, and its gradient 49, 5.4 TB/s (in part from the last
// cache). Few or short rows are a chain of load, sum, join and logarithms: 16 x 65536
// f16 9.2; 331 x 20011 f32 10.6, gradient 14.5. Back to back in a graph: 331 x 20011
// f32 loss 9.0, loss and gradient 16; 2000 x 65536 f32 119 (4.4 TB/s) and 243 (4.3).
#include "logits_rows.h"
#include "rwkv7_kernels.h"

namespace rwkv7 {
namespace {

constexpr int kDistMaxK = kRowMaxThreads;
// Half a step of such an lse is a factor e and more of every p. Rows masked by their
// type's lowest value have one (bf16, f32: -3e38 / temperature, or -inf where that is past
// f32), and p as it fell, 0, 1 or infinite.
constexpr double kNoTeacher = -0x1p24;
constexpr double kLn2 = 0.69314718055994531, kLog2E = 1.4426950408889634;

struct DistillArgs {
  const void *logits;
  int64_t ld;
  int V, K;
  ExpScale sc;
  double a;
  const void *top_val;
  int val_fmt;
  const int64_t *top_idx;
  const float *lse;    // null: softmax over the entries
  const float *scale;  // upstream gradient of each row, null: scale0
  float scale0;
  float *loss;         // null: not wanted
  void *grad;          // null: not wanted
  int64_t grad_ld;
  int64_t row0;
};

struct Joined {
  float m, mrest;       // what the row's sum is about, and that without the entries' ids
  double S, Srest;      // sums about them
  double in_all;        // what a sum about mrest counts in one about m
  double W, tref;       // the teacher's mass about its reference
  double P, rest_t;
  bool mass;
};

struct DistillLds {
  u64 mine[kRowMaxThreads];  // of each thread's logits, bit 8 c + e for chunk c: those with an entry
  uint32_t tail;             // of the logits behind the eights
  int idx[kDistMaxK];        // of each thread's entry, -1 for none
  float z[kDistMaxK];        // its student logit
  // per wave: of the row's rest a logit and the sum about it, of the entries the
  // largest and the sum about that; the teacher's reference, mass, and
  // mass-weighted difference of its logarithms about that and the student's about
  // mtop
  float mrest[kMaxWaves], rest[kMaxWaves], mtop[kMaxWaves];
  double top[kMaxWaves], tref[kMaxWaves], tw[kMaxWaves], ta[kMaxWaves];
  bool whole;  // every id of the vocabulary has an entry
  Joined j;
  float f_rest;
  double f_top, ua;
};

template <int FMT, int THREADS>
RWKV7_DEV void zero_row(char *dst, int V) {
  const float zero[kRowChunk] = {};
#pragma unroll 1
  for (uint32_t b = threadIdx.x; b < (uint32_t)V / kRowChunk; b += THREADS) store_chunk<FMT>(dst, b, zero);
  if (threadIdx.x < V % kRowChunk) store_logit<FMT>(dst, V / kRowChunk * kRowChunk + threadIdx.x, 0.f);
}

// The least mass outside the ids that counts: half a step of the f32 Lt, which rounding
// alone can take from 1 (P = exp(-half a step) of a teacher whose every logit with
// any mass is listed), but no less than 2^-20, the half step of 16 <= |Lt| < 32. (With
// 2^-20 for all, an Lt of 200 made a rest of up to 8e-6, and a student with 1e-30 outside
// the ids paid 5e-4 for it.)
RWKV7_DEV double least_rest(double lse) {
  int ex;
  (void)frexpf((float)lse, &ex);
  return fmax(0x1p-20, ldexp(1.0, ex - 25));
}

// The waves' parts joined by one wave, one a lane. Logarithms and the teacher's
// references are to base 2, but lse.
template <int WAVES>
RWKV7_DEV Joined join(const DistillArgs &g, const DistillLds &s, int lane, double lse) {
  Joined j;
  const float mr = lane < WAVES ? s.mrest[lane] : -kInf, mt = lane < WAVES ? s.mtop[lane] : -kInf;
  j.mrest = uniform_f(wave_max(mr));
  const float mtop = wave_max(mt);
  j.m = uniform_f(fmaxf(j.mrest, mtop));
  j.Srest = uniform_d(wave_sum_d(lane < WAVES ? (double)s.rest[lane] * g.sc.part(mr, j.mrest) : 0.0));
  const double Stop = wave_sum_d(lane < WAVES ? s.top[lane] * g.sc.shift(mt, mtop) : 0.0);
  j.in_all = uniform_d(g.sc.part_of_exact(j.mrest, j.m));
  j.S = uniform_d(j.Srest * j.in_all + Stop * g.sc.shift(mtop, j.m));
  if (!(j.m > -kInf)) j.S = __builtin_nan("");  // no finite logit at all
  const int tws = (g.K + kWave - 1) / kWave;
  double W = lane < tws ? s.tw[lane] : 0.0;
  j.tref = 0.0;
  if (!g.lse) {
    const double tr = lane < tws ? s.tref[lane] : -__builtin_inf();
    j.tref = uniform_d(wave_max_d(tr));
    W *= tr > -__builtin_inf() ? exp2_d(tr - j.tref) : 0.0;
  }
  j.W = uniform_d(wave_sum_d(W));
  if (lse != lse) j.W = lse;  // (also where all entries are -inf)
  j.P = j.W, j.rest_t = 0.0;
  if (g.lse) {
    j.rest_t = uniform_d(1.0 - j.W);
    if (j.rest_t < least_rest(lse) || s.whole) j.rest_t = 0.0;
  } else {
    j.P = j.W == j.W ? 1.0 : j.W;
  }
  j.mass = g.lse ? !(lse <= kNoTeacher) : j.W != 0.0;  // (NaN: the row's loss is NaN)
  return j;
}

RWKV7_DEV void put_loss(const DistillArgs &g, const DistillLds &s, const Joined &j, int lane, int64_t row) {
  const int tws = (g.K + kWave - 1) / kWave;
  // sum p (log p - log q), in log q = k (z - m) - log S, without log S
  double A = 0.0;
  if (lane < tws) {
    const double tr = s.tref[lane], f = g.lse ? 1.0 : tr > -__builtin_inf() ? exp2_d(tr - j.tref) : 0.0;
    const double up = (g.lse ? 0.0 : tr - j.tref) - g.sc.k * ((double)ExpScale::ref(s.mtop[lane]) - (double)j.m);
    A = s.tw[lane] != 0.0 ? f * (s.ta[lane] + s.tw[lane] * up) : 0.0;
  }
  A = wave_sum_d(A);
  const double S = log2_d(j.S);
  double loss;
  if (g.lse) {
    loss = A + j.W * S;
    if (j.rest_t > 0.0)
      loss += j.rest_t * (log2_d(j.rest_t) - (g.sc.k * ((double)j.mrest - (double)j.m) + (g.sc.off(j.mrest) + log2_d(j.Srest)) - S));
  } else {
    loss = A * rcp_d(j.W) - log2_d(j.W) + S;
  }
  if (!j.mass) loss = 0.0;
  if (lane == 0) g.loss[row] = (float)(kLn2 * loss);
}

template <int FMT, int THREADS, bool LOSS, bool GRAD>
__global__ __launch_bounds__(THREADS, FMT == 1 ? 4 : 8) void distill_kernel(DistillArgs g) {
  __shared__ DistillLds s;
  constexpr int kWaves = THREADS / kWave;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, V = g.V;
  const uint32_t n8 = (uint32_t)V / kRowChunk;
  const int64_t row = g.row0 + blockIdx.x;
  const char *src = static_cast<const char *>(g.logits) + row * g.ld * kLogitBytes<FMT>;
  char *dst = GRAD ? static_cast<char *>(g.grad) + row * g.grad_ld * kLogitBytes<FMT> : nullptr;
  const float up = GRAD ? (g.scale ? g.scale[row] : g.scale0) : 0.f;

  // the teacher's entry of this thread
  const int64_t id64 = t < g.K ? g.top_idx[row * g.K + t] : -1;
  const bool there = id64 >= 0 && id64 < V;
  const int id = there ? (int)id64 : -1;
  s.mine[t] = 0;
  if (t == 0) s.tail = 0u;
  const bool some = __syncthreads_or(there);
  if (!some) {
    if (LOSS && t == 0) g.loss[row] = 0.f;
    if (GRAD) zero_row<FMT, THREADS>(dst, V);
    return;
  }
  Chunk<FMT> x[kRowChunks];
  load_row<THREADS>(x, src, n8);
  const int tail = t < V % kRowChunk ? (int)n8 * kRowChunk + t : -1;  // this thread's logit behind the eights
  float xt = tail >= 0 ? load_logit<FMT>(src, tail) : -kInf;
  const float tv = there ? load_logit_rt(g.top_val, row * g.K + t, g.val_fmt) : -kInf;
  const float zv = there ? load_logit<FMT>(src, id) : -kInf;
  const double lse = uniform_d(g.lse ? (double)g.lse[row] : 0.0);

  // mark the ids; `first`: this entry stands for its id. (Id and logit wait in LDS
  // for the gradient: nothing is held beside the row.)
  s.idx[t] = id;
  if (GRAD) s.z[t] = zv;
  bool first = there;
  if (there) {
    const uint32_t b = (uint32_t)id / kRowChunk, bit = b / THREADS * kRowChunk + id % kRowChunk;
    uint32_t *word = b < n8 ? reinterpret_cast<uint32_t *>(&s.mine[b % THREADS]) + bit / 32 : &s.tail;
    const uint32_t own = b < n8 ? 1u << bit % 32 : 1u << id % kRowChunk;
    first = !(atomicOr(word, own) & own);
  }
  const bool twice = __syncthreads_or(there && !first);
  if (twice) {  // the same id in several entries: the lowest stands for it
    __syncthreads();
    first = there;
#pragma unroll 1
    for (int k = 0; k < t; ++k) first = first && s.idx[k] != id;
  }
  if (g.K >= V) {  // (else some id is left over)
    const bool whole = __syncthreads_count(first) == V;
    if (t == 0) s.whole = whole;
  } else if (t == 0) {
    s.whole = false;
  }

  // this thread's part of the row without the entries' ids
  const u64 mine = s.mine[t];
  if (tail >= 0 && (s.tail >> t) & 1u) xt = -kInf;
  const bool entries = wv * kWave < g.K;  // this wave has entries
  const float mtop = entries ? wave_max(zv) : -kInf;
  float m;
  const float sum = sum_row<THREADS, false, !GRAD>(x, src, n8, xt, g.sc, m, [&](int c, Chunk<FMT> &y) {
    const uint32_t marked = (uint32_t)(mine >> (kRowChunk * c)) & 255u;
    if (marked) y.remove(marked);
  });

  // the entries in 64 bits and powers of two: the student's about their largest,
  // the teacher's about its lse or the wave's largest (a gradient's q - p is what
  // is left of the two). Differences come before the factor: a product less a rounded
  // one, which the compiler joins in one fma, is what the rounding took, 1e22 at the
  // lowest value of f32, and a row of that alone had p of 2^1e22.
  const double k2 = g.sc.k;
  double tref = 0.0, w = 0.0;
  if (entries) {
    const double zk = k2 * ((double)zv - (double)ExpScale::ref(mtop));  // (NaN stays NaN)
    const double top = wave_sum_d(first ? zk == zk ? exp2_d(zk) : zk : 0.0);
    double y;  // (NaN stays NaN)
    if (g.lse) {
      y = kLog2E * (g.a * (double)tv - lse);
    } else {
      const double most = (double)wave_max(tv);
      tref = k2 * most;
      y = k2 * ((double)tv - most);
    }
    w = there && tv != -kInf ? (y == y ? exp2_d(y) : y) : 0.0;
    const double ta = w != 0.0 ? w * (y - zk) : 0.0;
    const double ws = wave_sum_d(w), as = wave_sum_d(ta);
    if (lane == 0) s.tref[wv] = tref, s.tw[wv] = ws, s.ta[wv] = as, s.top[wv] = top;
    if (GRAD) s.mine[t] = __builtin_bit_cast(u64, w);  // (the marks are used up)
  }
  if (lane == 0) s.mrest[wv] = m, s.rest[wv] = sum, s.mtop[wv] = mtop;
  if (!entries && lane == 0) s.top[wv] = 0.0;
  __syncthreads();

  if (wv == 0) {
    const Joined j = join<kWaves>(g, s, lane, lse);
    if (!GRAD) {
      put_loss(g, s, j, lane, row);
      return;
    }
    // d loss / d z, scaled: f_rest e for the rest, f_top e - ua p for the entries
    const double ua = j.mass ? (double)up * g.a : 0.0, all = ua * (j.P + j.rest_t) * rcp_d(j.S);
    if (lane == 0) {
      s.j = j;
      s.ua = ua;
      s.f_top = all;
      s.f_rest = (float)(all * j.in_all - (j.rest_t > 0.0 && j.Srest > 0.0 ? ua * j.rest_t * rcp_d(j.Srest) : 0.0));
    }
  }
  if (!GRAD) return;
  __syncthreads();
  if (s.ua == 0.0) {  // a row that counts for nothing: zeros, not 0 * NaN
    zero_row<FMT, THREADS>(dst, V);
  } else {
    const float f_rest = uniform_f(s.f_rest);
    g.sc.with(s.j.mrest, [&](auto e2, auto far) {
#pragma unroll
      for (int c = 0; c < kRowChunks; ++c) {
        if (c > 0 && c * THREADS >= (int)n8) break;
        float f[kRowChunk];
        x[c].template get<decltype(far)::value>(f);
#pragma unroll
        for (int e = 0; e < kRowChunk; ++e) f[e] = f_rest * e2(f[e]);
        const uint32_t b = c * THREADS + t;
        if ((c + 1) * THREADS <= n8) store_chunk<FMT>(dst, b, f);
        else if (b < n8) store_chunk<FMT>(dst, b, f);
      }
      if (t < V % kRowChunk) store_logit<FMT>(dst, (int)n8 * kRowChunk + t, f_rest * e2(xt));
    });
    double pk = 0.0;
    if (wv * kWave < g.K) {
      pk = __builtin_bit_cast(double, s.mine[t]);
      if (!g.lse) pk *= exp2_d(s.tref[wv] - s.j.tref) * rcp_d(s.j.W);
    }
    if (twice) {
      s.mine[t] = __builtin_bit_cast(u64, s.idx[t] >= 0 ? pk : 0.0);
      __syncthreads();
      double sum = 0.0;
#pragma unroll 1
      for (int k = 0; first && k < g.K; ++k) sum += s.idx[k] == s.idx[t] ? __builtin_bit_cast(double, s.mine[k]) : 0.0;
      pk = sum;
    }
    __syncthreads();  // the row's own stores come before the entries'
    if (first) {
      const double zk = g.sc.k * ((double)s.z[t] - (double)s.j.m);  // (NaN stays NaN)
      store_logit<FMT>(dst, s.idx[t], (float)(s.f_top * (zk == zk ? exp2_d(zk) : zk) - s.ua * pk));
    }
  }
  if (LOSS && wv == 0) put_loss(g, s, s.j, lane, row);
}

template <int FMT, int THREADS>
void launch_t(const DistillArgs &g, int N, hipStream_t st) {
  if (g.grad && g.loss) distill_kernel<FMT, THREADS, true, true><<<N, THREADS, 0, st>>>(g);
  else if (g.grad) distill_kernel<FMT, THREADS, false, true><<<N, THREADS, 0, st>>>(g);
  else distill_kernel<FMT, THREADS, true, false><<<N, THREADS, 0, st>>>(g);
}

template <int FMT>
void launch_f(const DistillArgs &g, int N, hipStream_t st) {
  // one entry a thread
  const int T = row_threads(g.V) > g.K ? row_threads(g.V) : g.K <= 256 ? 256 : g.K <= 512 ? 512 : 1024;
  if (T == 256) launch_t<FMT, 256>(g, N, st);
  else if (T == 512) launch_t<FMT, 512>(g, N, st);
  else launch_t<FMT, 1024>(g, N, st);
}

}  // namespace
}  // namespace rwkv7

extern "C" int rwkv7_distill(const void *logits, int32_t logits_dtype, int64_t ld, int32_t N, int32_t V,
                             const void *top_val, int32_t val_dtype, const int64_t *top_idx, int32_t K, const float *lse,
                             double temperature, const float *scale, float scale0, float *loss, void *grad,
                             int64_t grad_ld, void *stream) {
  using namespace rwkv7;
  if (!logits || !top_val || !top_idx || (!loss && !grad)) return RWKV7_EINVAL;
  if (logits_dtype < 0 || logits_dtype > 2 || val_dtype < 0 || val_dtype > 2) return RWKV7_EINVAL;
  if (!(temperature > 0.0) || temperature > 1e30 || temperature < 1e-30) return RWKV7_EINVAL;
  if (N < 1 || V < 1 || V > kRowMaxV || K < 1 || K > kDistMaxK || ld < V || (grad && grad_ld < V)) return RWKV7_ESHAPE;
  const double a = 1.0 / temperature;
  DistillArgs g = {logits, ld, V, K, ExpScale::of(a), a, top_val, val_dtype, top_idx, lse, scale, scale0, loss, grad, grad_ld, 0};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  for (; g.row0 < N; g.row0 += kLaunchRows) {
    const int n = N - g.row0 < kLaunchRows ? (int)(N - g.row0) : kLaunchRows;
    switch (logits_dtype) {
      case 0: launch_f<0>(g, n, st); break;
      case 1: launch_f<1>(g, n, st); break;
      default: launch_f<2>(g, n, st); break;
    }
    RWKV7_CHECK_LAUNCH();
  }
  return RWKV7_OK;
}
