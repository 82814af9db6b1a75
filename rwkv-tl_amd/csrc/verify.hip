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
// as much as one 32-bit fma on this machine, so an exponential of 12 of them
// and 6 others takes about as long as reading its logit.
//
// NaN counts as -inf (never drawn, never accepted). A drafted id outside the
// vocabulary is rejected, a row without a finite logit has no probability: its
// drafted token is rejected, and the next token falls to 0 if nothing is left to
// draw from.
//
// verify_stats_kernel: a slice of a row per workgroup: the sum of its
//   exponentials, about 0 or (where that comes out far from 1) about its largest
//   logit, for target rows also of each 512 logits (greedy: largest logit and its
//   first id). 8192 logits a workgroup, so that one sequence of four drafts already
//   has 72 of them. 96 sequences of up to 7 drafts x 65536 bf16, 830 rows that count:
//   41 us (109 MB, 2.6 TB/s), the vector units busy 86 % of it at 1.86 GHz with 19.6
//   instructions a logit, 12 of them 64-bit. 16 x 8 f16 10.2, 1 x 4 4.1.
// verify_draw_kernel: 2048 logits (large batches: 8192) of each sequence's decisive
//   row: every workgroup joins the sums of its sequence's rows and decides how many tokens are
//   accepted; the sums of max(p - q, 0) over each 512 of its logits; the last
//   workgroup of a sequence to finish (the only one that stays, where all tokens
//   are accepted) finds the 512 in which the running sum crosses, and in them the
//   token, by one wave. (As a launch of its own this draw took 3 us more of a call's
//   chain and 2 of its host time.) A chain of seven dependent trips to memory and
//   three prefixes: 10.0 us for one sequence, 12.0 for 16, 19.3 for 96. Both
//   kernels back to back in a graph, 1 x 4 / 16 x 8 / 96 x 7: 12.6 / 21.7 / 59 us, and of
//   drafts without a draw, whose rows are half as many, 11.0 / 19.3 / 39.
// verify_greedy_kernel: a wave per sequence, 3.6 us, most of it the launch.
#include "logits_rows.h"
#include "rwkv7_kernels.h"

namespace rwkv7 {
namespace {

constexpr int kVerThreads = 256;
constexpr int kVerWaves = kVerThreads / kWave;
constexpr int kVerChunks = 4;
constexpr int kSlice = kVerThreads * kVerChunks * kRowChunk;  // 8192 logits
constexpr int kMaxSlices = kRowMaxV / kSlice;                 // 8
constexpr int kBlocks = kVerChunks * kVerWaves;               // of 512 logits in a slice, in order
constexpr int kDrawE = 3;                                     // block sums per lane of the draw
// Workgroups of the draw, one per 2048 logits, above which each takes four times as
// many: all of a sequence's decide the same, which then counts for more than a
// longer chain. (Calls of 65536 bf16 logits, one / four: 24 x 5 21.7 / 22.5 us, 48 x 5
// 28.4 / 30.4, 64 x 7 41.9 / 38.9, 96 x 7 56.8 / 55.0.)
constexpr int kDrawWide = 1792;
constexpr int kVerMaxK = kWave - 1;                           // a lane per drafted token and one for the row behind them
static_assert(kMaxSlices * kBlocks + 1 <= kDrawE * kWave, "the draw's wave holds every block's sum, and the last logits'");

// What is known of a sequence once its rows are summed.
struct Decision {
  int n, rejected;  // accepted tokens; whether the next was drafted and rejected
  int x;            // the rejected token of a one-hot draft, else -1
  float mp, mq;     // what the sums of the row behind the accepted tokens are about, of target and draft
  double ip, iq;    // 1 / those sums, 0 for an empty row or none
};

struct VerifyArgs {
  const void *target, *draft;  // draft null: one-hot
  int64_t tb, tr, db, dr;      // strides of a sequence and of a row, in elements
  const int64_t *tok;
  const float *u;
  const int64_t *len;          // null: K
  int B, K, V, G;              // G slices of a row
  double kt, kd;               // log2(e) / temperature of target and draft; kt <= 0: greedy
  float endt, endd;            // 1000 / those
  int64_t *out, *accepted;
  // workspace
  double *sum;                 // [rows][G] sum of exponentials about m (greedy: first id of the largest)
  double *block;               // [B (K + 1)][G kBlocks + 1] the same by blocks; last: the logits behind the eights
  double *rest;                // [B][G kBlocks + 1] sums of max(p - q, 0)
  int *done;                   // [B] workgroups that have stored theirs
  float *m;                    // [rows][G] what a slice's sums are about: 0 or its largest logit (greedy: that); rows: B
                               // (K + 1) of the target, B K of the draft
};

// The exponentials of a row about m, 0 or its largest logit: 2^(k (x - m)), 1 at m,
// also at +inf; 0 for -inf and NaN.
struct Weight {
  float m;         // NaN: the row is empty
  double ref, k;
  RWKV7_DEV Weight(float largest, double k_)
      : m(largest > -kInf ? largest : __builtin_nanf("")), ref(largest > -kInf ? (double)largest : 0.0), k(k_) {}
  // (the difference first: k x - k m would lose it at the types' lowest values)
  RWKV7_DEV double operator()(float x) const { return x == m ? 1.0 : exp2_d(((double)x - ref) * k); }
};

// The same in bulk, about 0: 2^(k x), which 64 bits hold for |k x| up to 1000, so
// that a slice needs no pass for its largest. The power's whole part is added to
// the exponent's bits as it stands in the low word of k x + 1.5 2^52. Logits
// outside the range are moved to its ends: a sum over kMuch may hold some from
// above, and a slice from kLeast down is summed more exactly too: either is summed
// again about its largest. One moved up from below counts as 2^-1000, 512 of them as
// 2^-991, which is at most 2^-591 of a row that is summed about 0: a block whose share
// of what is drawn from is under kNoShare counts for nothing, so that no token is drawn
// whose logit is -inf or NaN. (Shares, not sums: of a row with a sum of 2^-145, -100 its
// largest logit, blocks of masked tokens alone were 2^-846 of the whole, more than a
// bound for sums of 2^-900, and u = 0 fell to their first.)
constexpr double kLeast = 0x1p-400, kNoShare = 0x1p-580, kMuch = 0x1p999;
struct BulkWeight {
  float end;  // 1000 / k
  double k;
  RWKV7_DEV double operator()(float x) const {
    const double d = (double)__builtin_amdgcn_fmed3f(x, -end, end), magic = 0x1.8p52;  // (NaN: -end)
    const double t = fma(d, k, magic), f = fma(d, k, magic - t);
    const u64 p = __builtin_bit_cast(u64, exp2_frac(f));
    uint32_t high = (uint32_t)(p >> 32);
    // (in assembly: the compiler makes a 64-bit addition of it, with three moves)
    asm("v_lshl_add_u32 %0, %1, 20, %0" : "+v"(high) : "v"((uint32_t)__builtin_bit_cast(u64, t)));
    return __builtin_bit_cast(double, (u64)(uint32_t)p | ((u64)high << 32));
  }
};

// A lane's four values summed over the wave, value l & 3 on lane l: lanes trade
// halves of the values before they add, 37 instructions for what takes four
// wave_sum_d 100.
constexpr int kDppRor4 = 0x124, kDppRor8 = 0x128;  // lane i <- i - 4, i - 8 within each 16
template <int CTRL>
RWKV7_DEV double trade_d(double even, double odd, bool is_odd) {
  return (is_odd ? odd : even) + dpp_d<CTRL>(is_odd ? even : odd);
}
RWKV7_DEV double wave_sums_d(const double (&v)[4]) {
  const int lane = threadIdx.x & (kWave - 1);
  double q = trade_d<kDppXor2>(trade_d<kDppXor1>(v[0], v[1], lane & 1), trade_d<kDppXor1>(v[2], v[3], lane & 1), lane & 2);
  q += dpp_d<kDppRor4>(q);
  q += dpp_d<kDppRor8>(q);
  auto rows = [&](auto swap) {  // rows of 16, then of 32 lanes
    const u64 u = __builtin_bit_cast(u64, q);
    const auto lo = swap((uint32_t)u), hi = swap((uint32_t)(u >> 32));
    q = __builtin_bit_cast(double, (u64)lo[0] | ((u64)hi[0] << 32)) + __builtin_bit_cast(double, (u64)lo[1] | ((u64)hi[1] << 32));
  };
  rows([](uint32_t w) { return __builtin_amdgcn_permlane16_swap(w, w, false, false); });
  rows([](uint32_t w) { return __builtin_amdgcn_permlane32_swap(w, w, false, false); });
  return q;
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
  __shared__ float s_m[kVerWaves];
  __shared__ double s_sum[kVerWaves];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, V = a.V, g = blockIdx.x;
  const int r = blockIdx.y, nt = a.B * (a.K + 1);
  const bool tgt = r < nt;
  const int per = tgt ? a.K + 1 : a.K, rr = tgt ? r : r - nt, b = rr / per, i = rr - b * per;
  const int len = drafted(a, b);
  if (tgt && i == 0 && g == 0 && t == 0) a.done[b] = 0;
  if (i >= (tgt ? len + 1 : len)) return;  // a row that no decision looks at
  const void *row = tgt ? target_row<FMT>(a, b, i) : draft_row<FMT>(a, b, i);
  const uint32_t n8 = (uint32_t)V / kRowChunk;
  Chunk<FMT> x[kVerChunks];
#pragma unroll
  for (int c = 0; c < kVerChunks; ++c) x[c].load(row, (g * kVerChunks + c) * kVerThreads + t, n8);
  const int tail = g == a.G - 1 && t < V % kRowChunk ? (int)n8 * kRowChunk + t : -1;
  const float xt = tail >= 0 ? load_logit<FMT>(row, tail) : -kInf;
  auto largest = [&]() {  // of the slice (NaN loses)
    RowMax<FMT> most;
#pragma unroll
    for (int c = 0; c < kVerChunks; ++c) most.add(x[c]);
    float m = wave_max(fmaxf(most.value(), xt));
    if (lane == 0) s_m[wv] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kVerWaves; ++w) m = fmaxf(m, s_m[w]);
    return m;
  };
  if (GREEDY) {
    const float m = largest();
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
    const double first = -wave_max_d(-(double)at);
    if (lane == 0) s_sum[wv] = first;
    __syncthreads();
    if (t == 0) {
      a.m[(int64_t)r * a.G + g] = m;
      a.sum[(int64_t)r * a.G + g] = fmin(fmin(s_sum[0], s_sum[1]), fmin(s_sum[2], s_sum[3]));
    }
    return;
  }
  const double k = tgt ? a.kt : a.kd;
  const BulkWeight bulk{tgt ? a.endt : a.endd, k};
  double *block = tgt ? a.block + (int64_t)r * (a.G * kBlocks + 1) + g * kBlocks : nullptr;
  auto total = [&](auto weight) {  // of the slice, with its blocks' sums put down
    double own[kVerChunks];
#pragma unroll
    for (int c = 0; c < kVerChunks; ++c) {
      float f[kRowChunk];
      x[c].get(f);
      double q = 0.0, p = 0.0;
#pragma unroll
      for (int e = 0; e < kRowChunk; e += 2) q += weight(f[e]), p += weight(f[e + 1]);
      own[c] = q + p;
    }
    double sum = wave_sums_d(own);  // lane c: chunk c's
    if (block && lane < kVerChunks) block[lane * kVerWaves + wv] = sum;
    sum += dpp_d<kDppXor1>(sum);
    sum += dpp_d<kDppXor2>(sum);
    if (g == a.G - 1 && wv == 0) {  // the logits behind the eights
      const double q = wave_sum_d(tail >= 0 ? weight(xt) : 0.0);
      if (block && lane == 0) block[kBlocks] = q;
      sum += q;
    }
    if (lane == 0) s_sum[wv] = sum;
    __syncthreads();
    return (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
  };
  float m = 0.f;
  double sum = total(bulk);
  if (!(sum > kLeast && sum < kMuch)) {  // (the same in every thread)
    m = largest();
#pragma unroll
    for (int c = 0; c < kVerChunks; ++c) x[c].opaque();
    sum = total(Weight(m, k));
  }
  if (t == 0) {
    a.m[(int64_t)r * a.G + g] = m;
    a.sum[(int64_t)r * a.G + g] = sum;
  }
}

struct DecideLds {
  float m[2][kWave];
  double S[2][kWave];
  Decision d;
};

// How many of sequence b's tokens are accepted, by a workgroup: the rows' sums
// joined, a thread per slice, then a lane per drafted token.
template <int FMT>
RWKV7_DEV void decide(const VerifyArgs &a, int b, DecideLds &s) {
  const int t = threadIdx.x;
  // Every row's sums and every token, also those that the length leaves out
  // (their sums are not written): no load here waits for the length.
  float zp = -kInf, zq = -kInf, u = 0.f;
  int64_t x = -1;
  if (t < a.K) {
    x = a.tok[(int64_t)b * a.K + t];
    u = a.u[(int64_t)b * (a.K + 1) + t];
    if (x >= 0 && x < a.V) {
      zp = load_logit<FMT>(target_row<FMT>(a, b, t), x);
      if (a.draft) zq = load_logit<FMT>(draft_row<FMT>(a, b, t), x);
    } else {
      x = -1;
    }
  }
  const int len = drafted(a, b), rows = 2 * a.K + 1;
  for (int i = t; i < (a.draft ? rows : a.K + 1) * kMaxSlices; i += kVerThreads) {  // (whole groups of eight lanes)
    const int r = i / kMaxSlices, g = i % kMaxSlices, which = r > a.K, row = which ? r - a.K - 1 : r;
    const int64_t at = (which ? (int64_t)a.B * (a.K + 1) + (int64_t)b * a.K + row : (int64_t)b * (a.K + 1) + row) * a.G + g;
    const float mg = g < a.G ? a.m[at] : -kInf;
    const double sum = g < a.G ? a.sum[at] : 0.0;
    float m = mg;
    m = fmaxf(m, dpp<kDppXor1>(m));
    m = fmaxf(m, dpp<kDppXor2>(m));
    m = fmaxf(m, dpp<kDppHalfMirror>(m));
    double S = mg > -kInf ? sum * Weight(m, which ? a.kd : a.kt)(mg) : 0.0;
    S += dpp_d<kDppXor1>(S);
    S += dpp_d<kDppXor2>(S);
    S += dpp_d<kDppHalfMirror>(S);
    if (g == 0) s.m[which][row] = m, s.S[which][row] = S;
  }
  __syncthreads();
  if (t < kWave) {
    bool ok = false;
    if (t < len && x >= 0) {
      const double Sp = s.S[0][t], Sq = a.draft ? s.S[1][t] : 0.0;
      const double px = Sp > 0.0 ? Weight(s.m[0][t], a.kt)(zp) / Sp : 0.0;
      const double qx = !a.draft ? 1.0 : Sq > 0.0 ? Weight(s.m[1][t], a.kd)(zq) / Sq : 0.0;
      ok = px > 0.0 && (double)u * qx < px;
    }
    const int n = __ffsll((u64)~__ballot(ok)) - 1;  // (lane len is never ok)
    if (t == n) {
      const bool rejected = n < len;
      Decision d;
      d.n = n, d.rejected = rejected;
      d.x = rejected && !a.draft ? (int)x : -1;
      d.mp = s.m[0][n];
      d.ip = s.S[0][n] > 0.0 ? 1.0 / s.S[0][n] : 0.0;
      const bool soft = rejected && a.draft;
      d.mq = soft ? s.m[1][n] : 0.f;
      d.iq = soft && s.S[1][n] > 0.0 ? 1.0 / s.S[1][n] : 0.0;
      s.d = d;
    }
  }
  __syncthreads();
}

// max(p - q, 0); both products rounded, so that equal rows leave nothing.
RWKV7_DEV double over(double wp, double ip, double wq, double iq) {
#pragma clang fp contract(off)
  return fmax(wp * ip - wq * iq, 0.0);
}

// The same of one logit from the exponentials; id: its index.
struct Residual {
  Weight p, q;
  double ip, iq;
  int x;
  bool soft;
  RWKV7_DEV Residual(const VerifyArgs &a, const Decision &d, bool from_p)
      : p(d.mp, a.kt), q(d.mq, a.kd), ip(d.ip), iq(d.iq), x(from_p ? -1 : d.x), soft(!from_p && d.rejected && a.draft) {}
  RWKV7_DEV double operator()(float xp, float xq, int id) const {
    const double r = soft ? over(p(xp), ip, q(xq), iq) : p(xp) * ip;
    return id == x ? 0.0 : r;
  }
};

RWKV7_DEV double shfl_up_d(double x, int d) {
  const u64 v = __builtin_bit_cast(u64, x);
  const int lo = __shfl_up((int)(uint32_t)v, d), hi = __shfl_up((int)(uint32_t)(v >> 32), d);
  return __builtin_bit_cast(double, (u64)(uint32_t)lo | ((u64)(uint32_t)hi << 32));
}
// Inclusive prefix over the lanes.
RWKV7_DEV double wave_scan_d(double v) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const double o = shfl_up_d(v, d);
    if ((int)threadIdx.x >= d) v += o;
  }
  return v;
}

// The token behind the accepted ones, and the outputs, by one wave.
template <int FMT>
RWKV7_DEV void draw(const VerifyArgs &a, int b, const Decision &d) {
  const int lane = threadIdx.x, V = a.V, blocks = a.G * kBlocks + 1;
  const uint32_t n8 = (uint32_t)V / kRowChunk;
  const double u = (double)a.u[(int64_t)b * (a.K + 1) + a.K];
  const int64_t r = (int64_t)b * (a.K + 1) + d.n;
  // this lane's block sums of what is drawn from: p - q, or p itself
  double w[kDrawE];
  bool from_p = !d.rejected;
  if (d.rejected) {
#pragma unroll
    for (int e = 0; e < kDrawE; ++e) {
      // (device-scope, as they were stored: other workgroups' of this launch)
      w[e] = kDrawE * lane + e < blocks ? __hip_atomic_load(a.rest + (int64_t)b * blocks + kDrawE * lane + e, __ATOMIC_RELAXED,
                                                            __HIP_MEMORY_SCOPE_AGENT)
                                        : 0.0;
      if (!(w[e] > kNoShare)) w[e] = 0.0;
    }
    from_p = !(wave_sum_d((w[0] + w[1]) + w[2]) > 0.0);
  }
  if (from_p) {
    const Weight weight(d.mp, a.kt);
#pragma unroll
    for (int e = 0; e < kDrawE; ++e) {
      const int i = kDrawE * lane + e, g = min(i / kBlocks, a.G - 1);
      w[e] = i < blocks ? a.block[r * blocks + i] * (weight(a.m[r * a.G + g]) * d.ip) : 0.0;
      if (!(w[e] > kNoShare)) w[e] = 0.0;
    }
  }
  double own = (w[0] + w[1]) + w[2];
  double inc = wave_scan_d(own);
  const double goal = u * lane_value_d(inc, kWave - 1);
  // the first block in which the running sum exceeds the goal; none (u >= 1, or
  // rounding): the last one with any weight
  u64 over = __ballot(own > 0.0 && inc > goal);
  const u64 some = __ballot(own > 0.0);
  const bool none = over == 0;
  int token = 0;  // with nothing to draw from
  if (some) {
    const int who = none ? 63 - __clzll(some) : __ffsll(over) - 1;
    double base = inc - own;
    int e0 = -1;
#pragma unroll
    for (int e = 0; e < kDrawE; ++e) {
      const bool stop = none ? w[e] > 0.0 : e0 < 0 && w[e] > 0.0 && base + w[e] > goal;
      if (stop) e0 = e;
      else if (e0 < 0) base += w[e];
    }
    // By rounding the running sum may end just below the goal: then the last token of
    // the lane's last block with any weight, as where nothing exceeds the goal.
    const bool end = none || __builtin_amdgcn_readlane(e0, who) < 0;
    if (e0 < 0) {
#pragma unroll
      for (int e = 0; e < kDrawE; ++e)
        if (w[e] > 0.0) e0 = e;
    }
    const int blk = __builtin_amdgcn_readlane(kDrawE * lane + e0, who);
    base = lane_value_d(base, who);
    // its logits, eight a lane (behind the eights: one)
    const bool last = blk == blocks - 1;
    const int g = blk / kBlocks, c = blk % kBlocks / kVerWaves, wv = blk % kVerWaves;
    const uint32_t e8 = last ? n8 : (g * kVerChunks + c) * kVerThreads + wv * kWave + lane;
    const void *pr = target_row<FMT>(a, b, d.n);
    const Residual res(a, d, from_p);
    const void *qr = res.soft ? draft_row<FMT>(a, b, d.n) : pr;
    Chunk<FMT> xp, xq;
    xp.load(pr, e8, n8);
    xq.load(qr, e8, n8);
    float fp[kRowChunk], fq[kRowChunk];
    xp.get(fp);
    xq.get(fq);
    int i0 = (int)e8 * kRowChunk;
    if (last) {
      i0 += lane;
      fp[0] = i0 < V ? load_logit<FMT>(pr, i0) : -kInf;
      fq[0] = i0 < V ? load_logit<FMT>(qr, i0) : -kInf;
    }
    double v[kRowChunk];
    auto weigh = [&](auto of) {
      own = 0.0;
#pragma unroll
      for (int e = 0; e < kRowChunk; ++e) own += v[e] = of(e);
      return __ballot(own > 0.0);
    };
    u64 here = weigh([&](int e) { return res(fp[e], fq[e], i0 + e); });
    // Where p and q differ by their last bits, the block's sum, of bulk exponentials, may
    // be a rounding that these do not have: then by p, so that no masked token is drawn.
    if (!here) here = weigh([&](int e) { return res.p(fp[e]) * d.ip; });
    inc = wave_scan_d(own);
    over = end ? 0 : __ballot(own > 0.0 && base + inc > goal);
    const int lane2 = over ? __ffsll(over) - 1 : here ? 63 - __clzll(here) : 0;
    double acc = base + (inc - own);
    int at = -1, back = 0;
#pragma unroll
    for (int e = 0; e < kRowChunk; ++e) {
      acc += v[e];
      if (v[e] > 0.0) {
        back = e;
        if (at < 0 && over && acc > goal) at = e;
      }
    }
    token = __builtin_amdgcn_readlane(i0 + (at < 0 ? back : at), lane2);
  }
  if (lane <= a.K) a.out[(int64_t)b * (a.K + 1) + lane] = lane < d.n ? a.tok[(int64_t)b * a.K + lane] : lane == d.n ? token : -1;
  if (lane == 0) a.accepted[b] = d.n;
}

// CH: chunks of 2048 logits a workgroup.
template <int FMT, int CH>
__global__ __launch_bounds__(kVerThreads) void verify_draw_kernel(VerifyArgs a) {
  __shared__ DecideLds s;
  __shared__ bool s_last;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, V = a.V, g = blockIdx.x, b = blockIdx.y;
  decide<FMT>(a, b, s);
  const Decision d = s.d;
  if (!d.rejected) {
    if (g == 0 && wv == 0) draw<FMT>(a, b, d);
    return;
  }
  const void *pr = target_row<FMT>(a, b, d.n), *qr = a.draft ? draft_row<FMT>(a, b, d.n) : pr;
  const uint32_t n8 = (uint32_t)V / kRowChunk;
  const Residual res(a, d, false);
  double *block = a.rest + (int64_t)b * (a.G * kBlocks + 1);
  Chunk<FMT> xp[CH], xq[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint32_t e8 = (g * CH + c) * kVerThreads + t;
    xp[c].load(pr, e8, n8);
    xq[c].load(qr, e8, n8);
  }
  double own[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int id = ((g * CH + c) * kVerThreads + t) * kRowChunk;
    float fp[kRowChunk], fq[kRowChunk];
    xp[c].get(fp);
    xq[c].get(fq);
    double sum = 0.0;
    if (d.mp == 0.f && d.mq == 0.f) {
      const BulkWeight p{a.endt, a.kt}, q{a.endd, a.kd};
#pragma unroll
      for (int e = 0; e < kRowChunk; ++e) {
        const double r = res.soft ? over(p(fp[e]), d.ip, q(fq[e]), d.iq) : p(fp[e]) * d.ip;
        sum += id + e == d.x ? 0.0 : r;
      }
    } else {
#pragma unroll 1
      for (int e = 0; e < kRowChunk; ++e) sum += res(fp[e], fq[e], id + e);
    }
    own[c] = sum;
  }
  // stored past the caches of this XCD, acknowledged before the count goes up
  auto put = [&](int i, double v) { __hip_atomic_store(block + i, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  if constexpr (CH == kVerChunks) {
    const double sum = wave_sums_d(own);  // lane c: chunk c's
    if (lane < CH) put((g * CH + lane) * kVerWaves + wv, sum);
  } else {
    static_assert(CH == 1);
    const double sum = wave_sum_d(own[0]);
    if (lane == 0) put(g * kVerWaves + wv, sum);
  }
  if (g == (int)gridDim.x - 1 && wv == 0) {  // the logits behind the eights
    const int id = (int)n8 * kRowChunk + t;
    const double sum = wave_sum_d(id < V ? res(load_logit<FMT>(pr, id), load_logit<FMT>(qr, id), id) : 0.0);
    if (lane == 0) put(a.G * kBlocks, sum);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (t == 0)
    s_last = __hip_atomic_fetch_add(a.done + b, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
  __syncthreads();
  if (s_last && wv == 0) draw<FMT>(a, b, d);
}

// Greedy: one wave per sequence, a lane per drafted token.
__global__ __launch_bounds__(kWave) void verify_greedy_kernel(VerifyArgs a) {
  const int lane = threadIdx.x, b = blockIdx.x, len = drafted(a, b);
  int best = a.V;
  if (lane <= len) {
    const int64_t r = (int64_t)b * (a.K + 1) + lane;
    float m = -kInf;
#pragma unroll
    for (int s = 0; s < kMaxSlices; ++s) {
      const int64_t at = r * a.G + min(s, a.G - 1);
      const float v = a.m[at];
      const int id = (int)a.sum[at];
      if (v > m) m = v, best = id;
    }
    if (best >= a.V) best = 0;
  }
  const int64_t x = lane < a.K ? a.tok[(int64_t)b * a.K + lane] : -1;
  const bool ok = lane < len && x == best;
  const int n = __ffsll((u64)~__ballot(ok)) - 1;
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
  if (a.B * a.G * kVerChunks > kDrawWide) verify_draw_kernel<FMT, kVerChunks><<<dim3(a.G, a.B), kVerThreads, 0, st>>>(a);
  else verify_draw_kernel<FMT, 1><<<dim3(a.G * kVerChunks, a.B), kVerThreads, 0, st>>>(a);
  RWKV7_CHECK_LAUNCH();
  return RWKV7_OK;
}

int64_t al256(int64_t x) { return (x + 255) / 256 * 256; }

// The workspace's parts in a's pointers; returns its size.
int64_t verify_ws(VerifyArgs &a, char *p) {
  const int64_t rows = (int64_t)a.B * (2 * a.K + 1), blocks = a.G * kBlocks + 1;
  char *const p0 = p;
  auto take = [&](int64_t bytes) {
    char *q = p;
    p += al256(bytes);
    return q;
  };
  a.sum = reinterpret_cast<double *>(take(rows * a.G * 8));
  a.block = reinterpret_cast<double *>(take((int64_t)a.B * (a.K + 1) * blocks * 8));
  a.rest = reinterpret_cast<double *>(take(a.B * blocks * 8));
  a.done = reinterpret_cast<int *>(take((int64_t)a.B * 4));
  a.m = reinterpret_cast<float *>(take(rows * a.G * 4));
  return p - p0;
}

}  // namespace
}  // namespace rwkv7

extern "C" int64_t rwkv7_verify_workspace_bytes(int32_t B, int32_t K, int32_t V) {
  using namespace rwkv7;
  if (B < 1 || K < 0 || K > kVerMaxK || V < 1 || V > kRowMaxV) return 0;
  VerifyArgs a;
  a.B = B, a.K = K, a.G = slices(V);
  return verify_ws(a, nullptr);
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
  VerifyArgs a;
  a.target = target, a.draft = soft ? draft : nullptr;
  a.tb = target_b, a.tr = target_r, a.db = draft_b, a.dr = draft_r;
  a.tok = tokens, a.u = uniforms, a.len = lengths;
  a.B = B, a.K = K, a.V = V, a.G = slices(V);
  a.kt = greedy ? 0.0 : kLog2E / temperature;
  a.kd = soft ? kLog2E / draft_temperature : 0.0;
  a.endt = (float)(1000.0 / a.kt), a.endd = (float)(1000.0 / a.kd);  // (0: inf, not read)
  a.out = out, a.accepted = accepted;
  verify_ws(a, static_cast<char *>(workspace));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (logits_dtype) {
    case 0: return launch_verify<0>(a, st);
    case 1: return launch_verify<1>(a, st);
    default: return launch_verify<2>(a, st);
  }
}
