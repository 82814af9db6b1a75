// Rows of up to 65536 logits held in the registers of one workgroup, and the
// order and wave reductions that the operators on such rows share.
//
// A row in registers is read once however many passes its operator makes over it
// (maximum, sum, selection, gradient). 64 logits a thread is what that needs at
// 65536 logits and 1024 threads: 32 registers in 16 bits, of the 64 that two such
// workgroups on a CU leave each thread (f32: 64 of 128, one workgroup). Two matter:
// one loads while the other computes (loss and gradient of 4096 x 65536 bf16 5.0 TB/s;
// of 2000 x 65536 f32 4.3). With the 27 registers a thread that spilled at first, loss
// and gradient of the former took 302 us; without, 244.
#pragma once

#include "rwkv7_common.h"

namespace rwkv7 {

typedef unsigned long long u64;

constexpr float kInf = __builtin_inff();
constexpr int kRowChunk = 8;                         // logits a thread loads at a time
constexpr int kRowChunks = 8;                        // such chunks per thread
constexpr int kRowE = kRowChunk * kRowChunks;        // logits per thread
constexpr int kRowMaxThreads = 1024;
constexpr int kRowMaxV = kRowMaxThreads * kRowE;     // 65536
constexpr int kMaxWaves = kRowMaxThreads / kWave;

// Threads of a workgroup for rows of V logits: the fewest of 256, 512, 1024
// that hold them, so that short rows leave room for more workgroups per CU (with
// 1024 for 20011 bf16 logits: loss of 2000 rows 27 -> 35 us, of 250 7.5 -> 8.0).
inline int row_threads(int V) { return V <= 256 * kRowE ? 256 : V <= 512 * kRowE ? 512 : 1024; }

// Rows of one launch, a workgroup each: a grid has fewer than 2^32 threads.
constexpr int kLaunchRows = 1 << 21;

// Bytes per logit: FMT 0 half, 1 f32, 2 bfloat16.
template <int FMT>
constexpr int kLogitBytes = FMT == 1 ? 4 : 2;
inline int logit_bytes(int fmt) { return fmt == 1 ? 4 : 2; }

template <int FMT>
RWKV7_DEV float load_logit(const void *row, int64_t i) {
  if constexpr (FMT == 1) return static_cast<const float *>(row)[i];
  else return F16T<FMT == 2>::to_f(static_cast<const uint16_t *>(row)[i]);
}

RWKV7_DEV float load_logit_rt(const void *p, int64_t i, int fmt) {
  return fmt == 1 ? static_cast<const float *>(p)[i] : u16_to_f(static_cast<const uint16_t *>(p)[i], fmt == 2);
}

template <int FMT>
RWKV7_DEV void store_logit(void *row, int64_t i, float v) {
  if constexpr (FMT == 1) static_cast<float *>(row)[i] = v;
  else static_cast<uint16_t *>(row)[i] = F16T<FMT == 2>::from_f(v);
}

// Eight logits as they lie in memory: 16 bytes, or 32 in f32. Rows may start
// at any element (the copies become 16-byte accesses, which need no alignment
// here). A row is its whole eights, eight b on thread b % threads, and the up to
// seven logits behind them, one each on the first threads.
template <int FMT>
struct Chunk {
  static constexpr bool F32 = FMT == 1;
  static constexpr int kWords = F32 ? 8 : 4;
  uint32_t w[kWords];

  RWKV7_DEV void fill_absent() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = F32 ? 0xff800000u : FMT == 2 ? 0xff80ff80u : 0xfc00fc00u;  // -inf
  }
  RWKV7_DEV void load_whole(const void *row, uint32_t b) {
    __builtin_memcpy(w, static_cast<const char *>(row) + b * (uint32_t)(kRowChunk * kLogitBytes<FMT>), sizeof w);
  }
  // the b-th eight of a row with n8 whole ones, -inf past them
  RWKV7_DEV void load(const void *row, uint32_t b, uint32_t n8) {
    fill_absent();
    if (b < n8) load_whole(row, b);
  }
  // The compiler would otherwise keep a row's unpacked values from one pass to the
  // next, which the registers of the larger workgroups do not hold: between two
  // passes the chunks are made opaque.
  RWKV7_DEV void opaque() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) asm volatile("" : "+v"(w[i]));
  }
  // the eight as f32. FAR: by byte permutes, for the far arm of ExpScale::with: code
  // that both arms had alike would be moved before the branch, a row's worth.
  template <bool FAR = false>
  RWKV7_DEV void get(float (&f)[kRowChunk]) const {
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < kRowChunk; ++e) f[e] = __uint_as_float(w[e]);
    } else if constexpr (FAR && FMT == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(__builtin_amdgcn_perm(w[i], 0u, 0x05040c0cu));
        f[2 * i + 1] = __uint_as_float(__builtin_amdgcn_perm(w[i], 0u, 0x07060c0cu));
      }
    } else {
      F16T<FMT == 2>::to_f8(make_uint4(w[0], w[1], w[2], w[3]), f);
    }
  }
  // the logits whose bit is set in `bits` become -inf
  RWKV7_DEV void remove(uint32_t bits) {
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < kRowChunk; ++e)
        if ((bits >> e) & 1u) w[e] = 0xff800000u;
    } else {
      constexpr uint32_t ninf = FMT == 2 ? 0xff80u : 0xfc00u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if ((bits >> (2 * i)) & 1u) w[i] = (w[i] & 0xffff0000u) | ninf;
        if ((bits >> (2 * i + 1)) & 1u) w[i] = (w[i] & 0x0000ffffu) | (ninf << 16);
      }
    }
  }
};

// The largest of some chunks' logits, NaN left out: halves in pairs.
template <int FMT>
struct RowMax {
  float m = -kInf;
  RWKV7_DEV void add(const Chunk<FMT> &x) {
    float f[kRowChunk];
    x.get(f);
#pragma unroll
    for (int e = 0; e < kRowChunk; ++e) m = fmaxf(m, f[e]);
  }
  RWKV7_DEV float value() const { return m; }
};
template <>
struct RowMax<0> {
  half2v m = {(_Float16)-kInf, (_Float16)-kInf};
  RWKV7_DEV void add(const Chunk<0> &x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(half2v, x.w[i]));
  }
  RWKV7_DEV float value() const { return fmaxf((float)m[0], (float)m[1]); }
};

// A workgroup's row: whole eights without a comparison where all threads have one.
template <int THREADS, int FMT>
RWKV7_DEV void load_row(Chunk<FMT> (&x)[kRowChunks], const void *row, uint32_t n8) {
#pragma unroll
  for (int c = 0; c < kRowChunks; ++c) {
    const uint32_t b = c * THREADS + threadIdx.x;
    if ((c + 1) * THREADS <= n8) x[c].load_whole(row, b);
    else x[c].load(row, b, n8);
  }
}
template <int FMT>
RWKV7_DEV void opaque_row(Chunk<FMT> (&x)[kRowChunks]) {
#pragma unroll
  for (int c = 0; c < kRowChunks; ++c) x[c].opaque();
}

// Eight values as the b-th eight of a row.
template <int FMT>
RWKV7_DEV void store_chunk(void *row, uint32_t b, const float (&f)[kRowChunk]) {
  char *p = static_cast<char *>(row) + b * (uint32_t)(kRowChunk * kLogitBytes<FMT>);
  if constexpr (FMT == 1) {
    __builtin_memcpy(p, f, 32);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (uint32_t)F16T<FMT == 2>::from_f(f[2 * i]) | ((uint32_t)F16T<FMT == 2>::from_f(f[2 * i + 1]) << 16);
    __builtin_memcpy(p, w, 16);
  }
}

// Sums and maxima of doubles over the wave by lane permutes and readlanes, as
// common's float ones: no LDS and no address registers; the result is uniform.
template <int CTRL>
RWKV7_DEV double dpp_d(double v) {
  const u64 u = __builtin_bit_cast(u64, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (u64)lo | ((u64)hi << 32));
}
RWKV7_DEV double lane_value_d(double v, int lane) {
  const u64 u = __builtin_bit_cast(u64, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (u64)lo | ((u64)hi << 32));
}
// A value that every lane holds, kept in scalar registers.
RWKV7_DEV double uniform_d(double v) { return lane_value_d(v, 0); }
RWKV7_DEV float uniform_f(float v) { return lane_value(v, 0); }
RWKV7_DEV double wave_sum_d(double v) {
  v += dpp_d<kDppXor1>(v);
  v += dpp_d<kDppXor2>(v);
  v += dpp_d<kDppHalfMirror>(v);
  v += dpp_d<kDppMirror>(v);
  return (lane_value_d(v, 0) + lane_value_d(v, 16)) + (lane_value_d(v, 32) + lane_value_d(v, 48));
}
RWKV7_DEV double wave_max_d(double v) {
  v = fmax(v, dpp_d<kDppXor1>(v));
  v = fmax(v, dpp_d<kDppXor2>(v));
  v = fmax(v, dpp_d<kDppHalfMirror>(v));
  v = fmax(v, dpp_d<kDppMirror>(v));
  return fmax(fmax(lane_value_d(v, 0), lane_value_d(v, 16)), fmax(lane_value_d(v, 32), lane_value_d(v, 48)));
}
RWKV7_DEV float wave_max(float v) {
  v = fmaxf(v, dpp<kDppXor1>(v));
  v = fmaxf(v, dpp<kDppXor2>(v));
  v = fmaxf(v, dpp<kDppHalfMirror>(v));
  v = fmaxf(v, dpp<kDppMirror>(v));
  return fmaxf(fmaxf(lane_value(v, 0), lane_value(v, 16)), fmaxf(lane_value(v, 32), lane_value(v, 48)));
}

// 2^f for |f| <= 1/2 in 64 bits, to 1.1e-12: the polynomial of degree 8 that
// interpolates it at the Chebyshev points. exp2_d: 2^y, y clamped to -2000 from
// below (0 there; NaN too). Fewer instructions and registers than the library's
// exp, and nearer than any sum here needs.
RWKV7_DEV double exp2_frac(double f) {
  double p = 1.3255224883682684e-06;
  p = fma(p, f, 1.5310079402211905e-05);
  p = fma(p, f, 0.00015403455852430636);
  p = fma(p, f, 0.0013333450568000708);
  p = fma(p, f, 0.00961812915940259);
  p = fma(p, f, 0.055504109412059334);
  p = fma(p, f, 0.2402265069581299);
  p = fma(p, f, 0.6931471805459335);
  p = fma(p, f, 1.0);
  return p;
}
RWKV7_DEV double exp2_d(double y) {
  y = fmax(y, -2000.0);
  const double n = rint(y);
  return ldexp(exp2_frac(y - n), (int)n);
}
// 1 / x in 64 bits: the hardware's estimate and two Newton steps (0 -> inf).
RWKV7_DEV double rcp_d(double x) {
  double y = __builtin_amdgcn_rcp(x);
  const double e = fma(-x, y, 1.0);
  if (fabs(e) < 1.0) {  // (x is neither 0 nor infinite)
    y = fma(y, e, y);
    y = fma(y, fma(-x, y, 1.0), y);
  }
  return y;
}
// log2 in 64 bits (0 -> -inf, inf -> inf): the float logarithm of the mantissa and one
// Newton step of 2^y = x (its error of 1e-7 squared).
RWKV7_DEV double log2_d(double x) {
  int ex;
  const double f = frexp(x, &ex);
  const double y = (double)__builtin_amdgcn_logf((float)f);
  return fabs(y) < 2.0 ? (double)ex + (y + (f * exp2_d(-y) - 1.0) * 1.4426950408889634) : y;
}

template <bool B>
struct BoolConst {
  static constexpr bool value = B;
};

// exp(a x) over a row as powers of two about its largest logit m. Near 0 (|m kf|
// up to 2^20) about R, the float nearest to m kf: 2^(x kf - R), one fma an
// element; what R and kf lack of m k is common to the row and made up for by off()
// and in log2z(). Farther away R's rounding would be more than the logits'
// differences, and the difference is taken first: 2^((x - m) kf). So a row of any
// size, the types' lowest values included, has a sum of about 1 or more.
struct ExpScale {
  float kf;    // a log2(e) in float
  double k;    // the same in 64 bits
  static ExpScale of(double a) {
    const double k = a * 1.4426950408889634;
    return {(float)k, k};
  }
  // m: -inf for none, which any finite reference serves
  static RWKV7_DEV float ref(float m) { return m > -kInf ? m : 0.f; }
  RWKV7_DEV bool near(float m) const { return fabsf(ref(m) * kf) <= 1048576.f; }
  RWKV7_DEV float e_near(float x, float R) const { return __builtin_amdgcn_exp2f(fmaf(x, kf, -R)); }
  RWKV7_DEV float e_far(float x, float m) const { return __builtin_amdgcn_exp2f((x - m) * kf); }
  RWKV7_DEV float e(float x, float m) const {
    m = ref(m);
    return near(m) ? e_near(x, m * kf) : e_far(x, m);
  }
  // body(f, far), f(x) = e(x, m), with the choice made once (m wave-uniform)
  template <class Body>
  RWKV7_DEV void with(float m, Body body) const {
    m = uniform_f(ref(m));
    if (near(m)) {
      const float R = m * kf;
      body([&](float x) { return e_near(x, R); }, BoolConst<false>());
    } else {
      body([&](float x) { return e_far(x, m); }, BoolConst<true>());
    }
  }
  // what a sum about m has over one about m exactly, as a power of two
  RWKV7_DEV double off(float m) const {
    m = ref(m);
    return near(m) ? (double)(m * kf) - (double)m * (double)kf : 0.0;
  }
  // what a sum about m (0 for none) counts in one about a larger one, both exactly
  RWKV7_DEV double shift(float m, float larger) const {
    return m > -kInf ? exp2_d(((double)m - (double)larger) * k) : 0.0;
  }
  // the same of sums of e(), and of one of those in an exact one
  RWKV7_DEV double part(float m, float larger) const { return shift(m, larger) * exp2_d(off(m) - off(larger)); }
  RWKV7_DEV double part_of_exact(float m, float larger) const { return shift(m, larger) * exp2_d(off(m)); }
  // log2 of sum exp(a x) when the sum about m is S
  RWKV7_DEV double log2z(double S, float m) const { return (double)m * k + off(m) + log2_d(S); }
};

// Sum of exp(a x) over a wave's chunks, each handed to see(c, chunk) first, about a
// logit of its own finding, m: the largest of the wave's first chunks, so that the
// others are summed as they arrive and no pass goes before for the largest of
// all. That is at least m, and the sum 1 or more; where it runs over (a logit 41 a
// units above m), where the first chunks hold nothing, and far from 0, it is formed
// again about the largest: from memory, a chunk at a time, which is rare and holds
// nothing beside the row. KNOWN: m is the wave's largest already. SKIP: chunks that no
// thread has are left out (back to back, loss of 331 x 20011 f32 9.9 -> 9.2 us, top
// logits of 2000 x 20011 bf16 29.8 -> 26.8); where registers are short, in a kernel with a gradient, the
// branches cost a full row more (loss and gradient of 4096 x 65536 bf16 214 -> 225).
template <int THREADS, bool KNOWN, bool SKIP, int FMT, class See>
RWKV7_DEV float sum_row(Chunk<FMT> (&x)[kRowChunks], const void *src, uint32_t n8, float tail, const ExpScale &sc, float &m,
                        See see) {
  see(0, x[0]);
  if (!KNOWN) {
    RowMax<FMT> first;
    first.add(x[0]);
    m = wave_max(first.value());
  }
  const bool good = m > -kInf && sc.near(m);
  const float R = uniform_f(good ? m * sc.kf : 0.f);
  float sum = sc.e_near(tail, R);
#pragma unroll
  for (int c = 0; c < kRowChunks; ++c) {
    if (SKIP && c > 0 && c * THREADS >= (int)n8) break;
    if (c > 0) see(c, x[c]);
    float f[kRowChunk], q[kRowChunk];
    x[c].get(f);
#pragma unroll
    for (int e = 0; e < kRowChunk; ++e) q[e] = sc.e_near(f[e], R);
    sum += ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7]));
  }
  sum = wave_sum(sum);
  opaque_row(x);
  if (!(good && sum >= 0.5f && sum < 0x1p60f)) {  // (wave-uniform)
    auto each = [&](auto f) {
#pragma unroll 1
      for (int c = 0; c < kRowChunks; ++c) {
        Chunk<FMT> y;
        y.load(src, c * THREADS + threadIdx.x, n8);
        see(c, y);
        f(y);
      }
    };
    RowMax<FMT> most;
    each([&](const Chunk<FMT> &y) { most.add(y); });
    m = wave_max(fmaxf(most.value(), tail));
    sum = sc.e(tail, m);
    each([&](const Chunk<FMT> &y) {
      float f[kRowChunk];
      y.get(f);
#pragma unroll
      for (int e = 0; e < kRowChunk; ++e) sum += sc.e(f[e], m);
    });
    sum = wave_sum(sum);
  }
  return sum;
}

}  // namespace rwkv7
