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
// there up. (From r = 17 of four maxima a lane; where a mask leaves a wave without
// r of them, by the waves that have 64.) The logits from the floor up are gathered
// in LDS, dealt to 256 bins of equal key ranges, and ranked by the bins before
// theirs and by comparison within their own. Where more than kCandMax pass (long
// ties), the k-th largest is found exactly by passes over the row that count keys
// by eight bits, and the last id that a tie admits likewise, so that just k are
// gathered.
//
// Why bins: ranked each against all, some 400 candidates took 4.7 us a row. Measured
// (kernel trace, us; a large copy moves 5.05 TB/s here): 4096 x 65536 bf16, k 200,
// 131-139, 3.9-4.1 TB/s: the vector units are busy 91 % of it with 13 instructions a
// logit (maxima, exponentials, comparisons). 509 x 65536 bf16, k 64, 20, 3.3 TB/s: one
// round of two rows a CU, each a chain of load, floor, sum, gather and ranking. One row
// 9.1; 257 x 20011 f32 12.5 (back to back in a graph 9.9); 2000 x 65536 f32, k 64, back
// to back 125, 4.2 TB/s.
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
  int64_t row0;
};

constexpr int kBins = 256;
constexpr int kGroups = 4;      // maxima a lane keeps: of its chunks c, c % 4
// Lowest bit of a floor that is decided: the formats' last, f32's to 2^-15 of a value.
template <int FMT>
constexpr int kFloorLow = FMT == 2 ? 16 : FMT == 0 ? 13 : 8;

struct TopLds {
  u64 cand[kCandMax];
  uint16_t dealt[kCandMax];
  float m[kMaxWaves], sum[kMaxWaves];
  uint32_t floor[kMaxWaves];
  int some[kMaxWaves];
  int bin[kBins], at[kBins];  // of each bin: its logits, and where its next one goes
  int n, digit, above;
};

// Order-preserving key of a logit: 1 for NaN, which comes behind -inf; 0 is none.
RWKV7_DEV uint32_t top_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 -> 0
  const uint32_t k = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return x == x ? k : 1u;
}
RWKV7_DEV float top_key_inv(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// The r-th largest of the N keys that each lane of the wave holds, rounded down
// to bit LOW; 0 when fewer than r are not 0.
template <int LOW, int N>
RWKV7_DEV uint32_t rth_key(const uint32_t (&key)[N], int r) {
  uint32_t fl = 0;
#pragma unroll 1
  for (int bit = 31; bit >= LOW; --bit) {
    const uint32_t c = fl | (1u << bit);
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += __popcll(__ballot(key[i] >= c));
    if (n >= r) fl = c;
  }
  return fl;
}

// Exclusive prefix over s.bin into s.at, by wave 0.
RWKV7_DEV void scan_bins(TopLds &s) {
  const int lane = threadIdx.x;
  if (lane >= kWave) return;
  int c[kBins / kWave], own = 0;
#pragma unroll
  for (int e = 0; e < kBins / kWave; ++e) own += c[e] = s.bin[kBins / kWave * lane + e];
  int inc = own;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int o = __shfl_up(inc, d);
    if (lane >= d) inc += o;
  }
  int at = inc - own;
#pragma unroll
  for (int e = 0; e < kBins / kWave; ++e) {
    s.at[kBins / kWave * lane + e] = at;
    at += c[e];
  }
}

// f(logit, id) for every logit of the row, from memory: the way of the long ties,
// of which nothing is held in registers beside the row.
template <int FMT, int THREADS, class F>
RWKV7_DEV void each_logit(const char *src, int V, F f) {
  const uint32_t n8 = (uint32_t)V / kRowChunk;
#pragma unroll 1
  for (uint32_t b = threadIdx.x; b < n8; b += THREADS) {
    Chunk<FMT> x;
    x.load(src, b, n8);
    float v[kRowChunk];
    x.get(v);
#pragma unroll
    for (int e = 0; e < kRowChunk; ++e) f(v[e], (int)b * kRowChunk + e);
  }
  const int tail = (int)n8 * kRowChunk + threadIdx.x;
  if (threadIdx.x < kRowChunk && tail < V) f(load_logit<FMT>(src, tail), tail);
}

// One digit of a radix selection: digit(key, id) is 0 .. 255, lowest first, or -1
// for what the digits before ruled out. Of the digits, the one that holds the
// `need`-th is returned, and need less those before it.
template <int FMT, int THREADS, class D>
RWKV7_DEV int select_digit(const char *src, int V, int &need, TopLds &s, D digit) {
  const int t = threadIdx.x;
  __syncthreads();
  if (t < kBins) s.bin[t] = 0;
  __syncthreads();
  each_logit<FMT, THREADS>(src, V, [&](float v, int id) {
    const int d = digit(top_key(v), id);
    if (d >= 0) atomicAdd(&s.bin[d], 1);
  });
  __syncthreads();
  scan_bins(s);
  __syncthreads();
  if (t < kBins && s.at[t] < need && need <= s.at[t] + s.bin[t]) s.digit = t, s.above = s.at[t];
  __syncthreads();
  need -= s.above;
  return s.digit;
}

template <int FMT, int THREADS>
__global__ __launch_bounds__(THREADS, FMT == 1 ? 4 : THREADS == 256 ? 7 : 8) void top_kernel(TopArgs g) {
  __shared__ TopLds s;
  constexpr int kWaves = THREADS / kWave;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, V = g.V, k = g.k;
  const uint32_t n8 = (uint32_t)V / kRowChunk;
  const int64_t row = g.row0 + blockIdx.x;
  const char *src = static_cast<const char *>(g.logits) + row * g.ld * kLogitBytes<FMT>;
  Chunk<FMT> x[kRowChunks];
  load_row<THREADS>(x, src, n8);
  const int tail = t < V % kRowChunk ? (int)n8 * kRowChunk + t : -1;
  const float xt = tail >= 0 ? load_logit<FMT>(src, tail) : -kInf;
  if (t == 0) s.n = 0;
  if (t < kBins) s.bin[t] = 0;

  // the lane's largest, by groups of chunks (-inf also for none: a floor may be
  // too low, never too high)
  uint32_t own[kGroups];
  float m = -kInf;
  {
    RowMax<FMT> most[kGroups];
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) most[c % kGroups].add(x[c]);
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const float mg = i == 0 ? fmaxf(most[0].value(), xt) : most[i].value();
      own[i] = mg > -kInf ? top_key(mg) : 0u;
      m = fmaxf(m, mg);
    }
  }
  opaque_row(x);
  auto wave_floor = [&](int r) {
    const uint32_t lo = own[0] > own[1] ? own[0] : own[1], hi = own[2] > own[3] ? own[2] : own[3], one[1] = {lo > hi ? lo : hi};
    return r > 16 ? rth_key<kFloorLow<FMT>>(own, r) : rth_key<kFloorLow<FMT>>(one, r);
  };
  {
    const uint32_t fl = wave_floor((k + kWaves - 1) / kWaves);
    int some = 0;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) some += __popcll(__ballot(own[i] != 0u));
    if (lane == 0) s.floor[wv] = fl, s.some[wv] = some;
  }
  m = wave_max(m);
  const float sum = sum_row<THREADS, true, true>(x, src, n8, xt, g.sc, m, [](int, Chunk<FMT> &) {});
  if (lane == 0) s.m[wv] = m, s.sum[wv] = sum;
  __syncthreads();

  // the least floor, and the waves with 64 maxima or more, one a lane
  auto least_floor = [&]() {
    uint32_t f = lane < kWaves ? s.floor[lane] : ~0u;
#pragma unroll
    for (int d = 1; d < kMaxWaves; d <<= 1) {
      const uint32_t o = (uint32_t)__shfl_xor((int)f, d);
      f = o < f ? o : f;
    }
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)f);
  };
  uint32_t fl = least_floor();
  const int full = __popcll(__ballot(lane < kWaves && s.some[lane] >= kWave));
  if (fl == 0u && k <= full * kWave) {  // (block-uniform)
    const uint32_t f = s.some[wv] >= kWave ? rth_key<kFloorLow<FMT>>(own, (k + full - 1) / full) : ~0u;
    __syncthreads();
    if (lane == 0) s.floor[wv] = f;
    __syncthreads();
    fl = least_floor();
  }

  // (The counter's place is opaque: the compiler would otherwise join the lanes'
  // additions first, in twenty instructions for the one or two that there are.)
  int zero = 0;
  asm volatile("" : "+v"(zero));
  int *const next = &s.n + zero;
  auto gather = [&](float v, int id) {
    const int slot = atomicAdd(next, 1);
    if (slot < kCandMax) s.cand[slot] = ((u64)__float_as_uint(v) << 32) | (uint32_t)~id;
  };
  if (fl) {
    // by value: one comparison a logit, and no more where none of a wave's passes
    const float least = top_key_inv(fl);
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) {
      if (c > 0 && c * THREADS >= (int)n8) break;
      float v[kRowChunk];
      x[c].get(v);
#pragma unroll
      for (int e = 0; e < kRowChunk; ++e)
        if (v[e] >= least) gather(v[e], (c * THREADS + t) * kRowChunk + e);
    }
    if (tail >= 0 && xt >= least) gather(xt, tail);
  } else if (V <= kCandMax) {
    each_logit<FMT, THREADS>(src, V, gather);
  } else if (t == 0) {
    s.n = kCandMax + 1;
  }
  __syncthreads();
  int n = s.n;
  if (n > kCandMax) {  // block-uniform
    uint32_t kth = 0;
    int need = k;
#pragma unroll 1
    for (int sh = 24; sh >= 0; sh -= 8)
      kth |= (uint32_t)(255 - select_digit<FMT, THREADS>(src, V, need, s, [&](uint32_t key, int) {
               return ((key ^ kth) >> sh) >> 8 ? -1 : 255 - (int)((key >> sh) & 255u);
             })) << sh;
    int last = 0;  // the id of the need-th logit with that key
#pragma unroll 1
    for (int sh = 8; sh >= 0; sh -= 8)
      last |= select_digit<FMT, THREADS>(src, V, need, s, [&](uint32_t key, int id) {
                return key != kth || ((id ^ last) >> sh) >> 8 ? -1 : (id >> sh) & 255;
              }) << sh;
    if (t == 0) s.n = 0;
    if (t < kBins) s.bin[t] = 0;
    __syncthreads();
    each_logit<FMT, THREADS>(src, V, [&](float v, int id) {
      const uint32_t key = top_key(v);
      if (key > kth || (key == kth && id <= last)) gather(v, id);
    });
    __syncthreads();
    n = k;
  }

  // keys from `low` up, in bins of 2^shift, the highest first
  const float mm = wave_max(lane < kWaves ? s.m[lane] : -kInf);
  const uint32_t low = fl, range = max(top_key(mm), 1u) - low;
  const int shift = max(0, 24 - __clz((int)(range | 1u)));
  auto bin_of = [&](u64 c) { return kBins - 1 - (int)(((uint32_t)(c >> 32) - low) >> shift); };
#pragma unroll 1
  for (int i = t; i < n; i += THREADS) {  // (from here on by their keys)
    const u64 c = s.cand[i], own = ((u64)top_key(__uint_as_float((uint32_t)(c >> 32))) << 32) | (uint32_t)c;
    s.cand[i] = own;
    atomicAdd(&s.bin[bin_of(own)], 1);
  }
  __syncthreads();
  scan_bins(s);
  __syncthreads();
#pragma unroll 1
  for (int i = t; i < n; i += THREADS) {
    s.dealt[atomicAdd(&s.at[bin_of(s.cand[i])], 1)] = (uint16_t)i;
  }
  __syncthreads();
#pragma unroll 1
  for (int i = t; i < n; i += THREADS) {
    const u64 own = s.cand[s.dealt[i]];
    const int bin = bin_of(own), end = s.at[bin], first = end - s.bin[bin];
    if (first >= k) continue;
    int rank = first;
#pragma unroll 1
    for (int j = first; j < end; ++j) rank += s.cand[s.dealt[j]] > own;
    if (rank < k) {
      const int id = (int)~(uint32_t)own;
      g.idx[row * k + rank] = id;
      if constexpr (FMT == 1) static_cast<float *>(g.val)[row * k + rank] = reinterpret_cast<const float *>(src)[id];
      else static_cast<uint16_t *>(g.val)[row * k + rank] = reinterpret_cast<const uint16_t *>(src)[id];
    }
  }
  if (wv == 0) {
    const float mw = lane < kWaves ? s.m[lane] : -kInf;
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
  TopArgs g = {logits, ld, V, k, ExpScale::of(1.0 / temperature), val, idx, lse, 0};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  for (; g.row0 < N; g.row0 += kLaunchRows) {
    const int n = N - g.row0 < kLaunchRows ? (int)(N - g.row0) : kLaunchRows;
    switch (logits_dtype) {
      case 0: launch_top<0>(g, n, st); break;
      case 1: launch_top<1>(g, n, st); break;
      default: launch_top<2>(g, n, st); break;
    }
    RWKV7_CHECK_LAUNCH();
  }
  return RWKV7_OK;
}
