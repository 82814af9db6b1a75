// The k largest logits of each row, in order, with their ids, and the row's
// log-sum-exp: what a teacher hands on of its answers. One workgroup per row;
// the row stays in registers.
//
// Order: descending value (-0 is 0), ties by the lowest id, NaN behind
// everything. lse = log sum_j exp(a z_j), a = 1 / temperature, NaN if a logit
// is or is +inf, -inf if all are.
//
// Selection. Each wave finds the r-th largest of its lanes' maxima, r = ceil(k /
// waves), by ballots; the least of them over the waves is a floor that k logits
// of the row reach, and few more: each wave has r lanes with a logit from
// there up. The logits from the floor up are gathered in LDS and ranked by
// counting, for each, those that come before it. Where more than kCandMax pass
// (long ties; rows shorter than the workgroup's lanes do not reach that many),
// the k-th largest is found exactly, key bit by key bit over the whole row, and
// the last id that a tie admits likewise, so that just k are gathered.
#include "logits_rows.h"
#include "rwkv7_kernels.h"

namespace rwkv7 {
namespace {

constexpr int kTopMax = 256;    // largest k: waves of the smallest workgroup x 64 lanes' maxima
constexpr int kCandMax = 2048;  // logits gathered at most

struct TopArgs {
  const void *logits;
  int64_t ld;
  int V, k;
  ExpScale sc;
  void *val;
  int64_t *idx;
  float *lse;
};

struct TopLds {
  u64 cand[kCandMax];
  float m[kMaxWaves], sum[kMaxWaves];
  uint32_t floor[kMaxWaves];
  int count[kMaxWaves];
  int n;
};

// Order-preserving key of a logit: 1 for NaN, which comes behind -inf; 0 is none.
RWKV7_DEV uint32_t top_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 -> 0
  const uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return x == x ? k : 1u;
}

template <int FMT, int THREADS>
__global__ __launch_bounds__(THREADS, FMT == 1 ? 4 : 8) void top_kernel(TopArgs g) {
  __shared__ TopLds s;
  constexpr int kWaves = THREADS / kWave;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, V = g.V, k = g.k;
  const uint32_t n8 = (uint32_t)V / kRowChunk;
  const int64_t row = blockIdx.x;
  const char *src = static_cast<const char *>(g.logits) + row * g.ld * kLogitBytes<FMT>;
  Chunk<FMT> x[kRowChunks];
#pragma unroll
  for (int c = 0; c < kRowChunks; ++c) x[c].load(src, c * THREADS + t, n8);
  const int tail = t < V % kRowChunk ? (int)n8 * kRowChunk + t : -1;
  const float xt = tail >= 0 ? load_logit<FMT>(src, tail) : -kInf;
  if (t == 0) s.n = 0;

  // the lane's largest (-inf also for none: a floor may be too low, never too high)
  float m = xt;
#pragma unroll
  for (int c = 0; c < kRowChunks; ++c) {
    float f[kRowChunk];
    x[c].get(f);
#pragma unroll
    for (int e = 0; e < kRowChunk; ++e) m = fmaxf(m, f[e]);
  }
  {
    const uint32_t own = m > -kInf ? top_key(m) : 0u;
    const int r = (k + kWaves - 1) / kWaves;
    uint32_t fl = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 8; --bit) {  // (to 2^-15 of a value)
      const uint32_t c = fl | (1u << bit);
      if (__popcll(__ballot(own >= c)) >= r) fl = c;
    }
    if (lane == 0) s.floor[wv] = fl;
  }
  m = wave_max(m);
  const float R = ExpScale::ref(m);
  float sum = g.sc.e(xt, R);
#pragma unroll
  for (int c = 0; c < kRowChunks; ++c) {
    float f[kRowChunk];
    x[c].get(f);
    float q[kRowChunk];
#pragma unroll
    for (int e = 0; e < kRowChunk; ++e) q[e] = g.sc.e(f[e], R);
    sum += ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7]));
  }
  sum = wave_sum(sum);
  if (lane == 0) s.m[wv] = m, s.sum[wv] = sum;
  __syncthreads();

  uint32_t fl = s.floor[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) fl = min(fl, s.floor[w]);

  // f(key, id) for every logit that this thread holds
  auto each = [&](auto f) {
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) {
      const uint32_t b = c * THREADS + t;
      float v[kRowChunk];
      x[c].get(v);
      if (b < n8) {
#pragma unroll
        for (int e = 0; e < kRowChunk; ++e) f(top_key(v[e]), (int)(b * kRowChunk + e));
      }
    }
    if (tail >= 0) f(top_key(xt), tail);
  };
  auto gather = [&](uint32_t key, int id) {
    const int slot = atomicAdd(&s.n, 1);
    if (slot < kCandMax) s.cand[slot] = ((u64)key << 32) | (uint32_t)~id;
  };
  each([&](uint32_t key, int id) {
    if (key >= fl) gather(key, id);
  });
  __syncthreads();
  int n = s.n;
  if (n > kCandMax) {  // block-uniform
    auto count = [&](int own) {  // over the workgroup
      float c = wave_sum((float)own);  // (exact: at most 65 x 1024)
      __syncthreads();
      if (lane == 0) s.count[wv] = (int)c;
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) all += s.count[w];
      return all;
    };
    uint32_t kth = 0;
    int above = 0;  // logits with a key over kth
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = kth | (1u << bit);
      int own = 0;
      each([&](uint32_t key, int) { own += key >= c; });
      const int all = count(own);
      if (all >= k) kth = c;
      else above = all;
    }
    int last = 0;  // the lowest bound so that k - above ties have ids up to it
#pragma unroll 1
    for (int bit = 15; bit >= 0; --bit) {
      const int c = last + (1 << bit);  // are there enough below c?
      int own = 0;
      each([&](uint32_t key, int id) { own += key == kth && id < c; });
      if (count(own) < k - above) last = c;
    }
    __syncthreads();
    if (t == 0) s.n = 0;
    __syncthreads();
    each([&](uint32_t key, int id) {
      if (key > kth || (key == kth && id <= last)) gather(key, id);
    });
    __syncthreads();
    n = s.n;
  }

  for (int i = t; i < n; i += THREADS) {
    const u64 own = s.cand[i];
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) rank += s.cand[j] > own;
    if (rank < k) {
      const int id = (int)~(uint32_t)own;
      g.idx[row * k + rank] = id;
      if constexpr (FMT == 1) static_cast<float *>(g.val)[row * k + rank] = reinterpret_cast<const float *>(src)[id];
      else static_cast<uint16_t *>(g.val)[row * k + rank] = reinterpret_cast<const uint16_t *>(src)[id];
    }
  }
  if (wv == 0) {
    const float mw = lane < kWaves ? s.m[lane] : -kInf, mm = wave_max(mw);
    const double S = wave_sum_d(lane < kWaves ? (double)s.sum[lane] * g.sc.part(mw, mm) : 0.0);
    // (S is 0 where there is nothing but -inf)
    if (lane == 0) g.lse[row] = S == 0.0 ? -kInf : (float)(0.69314718055994531 * g.sc.log2z(S, mm));
  }
}

template <int FMT>
void launch_top(const TopArgs &g, int N, hipStream_t st) {
  switch (row_threads(g.V)) {
    case 256: top_kernel<FMT, 256><<<N, 256, 0, st>>>(g); break;
    case 512: top_kernel<FMT, 512><<<N, 512, 0, st>>>(g); break;
    default: top_kernel<FMT, 1024><<<N, 1024, 0, st>>>(g); break;
  }
}

}  // namespace
}  // namespace rwkv7

extern "C" int rwkv7_top_logits(const void *logits, int32_t logits_dtype, int64_t ld, int32_t N, int32_t V, int32_t k,
                                double temperature, void *val, int64_t *idx, float *lse, void *stream) {
  using namespace rwkv7;
  if (!logits || !val || !idx || !lse || logits_dtype < 0 || logits_dtype > 2) return RWKV7_EINVAL;
  if (!(temperature >= 1e-30 && temperature <= 1e30)) return RWKV7_EINVAL;
  if (N < 1 || V < 1 || V > kRowMaxV || ld < V || k < 1 || k > V || k > kTopMax) return RWKV7_ESHAPE;
  const TopArgs g = {logits, ld, V, k, ExpScale::of(1.0 / temperature), val, idx, lse};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (logits_dtype) {
    case 0: launch_top<0>(g, N, st); break;
    case 1: launch_top<1>(g, N, st); break;
    default: launch_top<2>(g, N, st); break;
  }
  RWKV7_CHECK_LAUNCH();
  return RWKV7_OK;
}
