// LayerNorm that keeps its statistics, and its gradients.
//
//   m = mean x, v = mean (x - m)^2, r = (v + eps)^-1/2, xh = (x - m) r, y = xh w + b
//   dx = r (g - mean g - xh mean(g xh)), g = dy w
//   dw = sum over rows of dy xh, db = sum over rows of dy
//
// Bytes bound both passes (x, y; x, dy, dx): a row stays in registers, one wave a row up
// to 2048 16-bit or 1024 32-bit channels (no barrier), a workgroup beyond. The forward pass
// has a wave (or workgroup) for each row, weight and bias from the CU's L1; a wave of the
// gradient takes several rows with the weight in registers.
//
// Measured (kernel trace, us; a large copy moves 5.09 TB/s here). Forward: 16384 x 2048 bf16 26.5
// (5.1 TB/s), f32 40, 4096 x 2048 9.9, f32 15, 1024 x 16384 19, f32 31, 7 x 2048 f16 3.5. Gradient and the joining of its
// workgroups' sums: 16384 x 2048 bf16 34.6 + 4.6 (5.1 TB/s with both), f32 75 + 4.8 (5.1),
// 4096 x 2048 bf16 13.0 + 3.9, f32 20 + 3.9, 331 x 1001 f32 5.9 + 3.8, 1024 x 16384 bf16 25.2 + 6.1, f32 48 + 6.4. Without
// the next row on its way the first took 45.8; with workgroups of 8 waves 39 (256 of them) or 44.
// The forward pass forced into the registers of 5, 6 or 8 waves a SIMD spills: 50, 70, 97.
//
// Statistics in 32 bits about a first mean, whose own rounding (what is left of the
// differences' mean) is taken out again: a row whose mean is many times its deviation
// keeps its differences. Where that rounding is more than about four times the deviation
// (rows of one value far from 0, or nearly), the differences are formed once more about
// the corrected mean. The gradient takes the rounding of the mean it is given out alike.
// Rows whose squares pass 2^100 are taken times 2^-72.
#include "row_parts.h"
#include "rwkv7_kernels.h"

namespace rwkv7 {
namespace {

constexpr int kNormMaxC = 16384;
constexpr float kFarScale = 0x1p-72f;

struct NormArgs {
  const void *x, *w, *b;
  int64_t ldx;
  void *y;
  float *mean, *rstd;  // null: not wanted
  int64_t N;
  int C;
  double eps;
};

struct NormGradArgs {
  const void *dy, *x, *w;
  int64_t lddy, ldx;
  const float *mean, *rstd;
  void *dx;
  float *part;  // [gridDim.x][2][C]: sums of dy xh and of dy
  int64_t N;
  int C;
};

// Sums over the WAVES waves of a row: K of them, in the same order for every wave. Two
// buffers in turn, so that one barrier a sum is enough.
template <int WAVES, int K>
struct RowReduce {
  float buf[2][WAVES][K];
};
template <int WAVES, int K>
RWKV7_DEV void row_reduce(RowReduce<WAVES, K> &s, int &turn, float (&v)[K]) {
  if constexpr (K == 2) {
    const float2 t = wave_sum2(v[0], v[1]);
    v[0] = t.x, v[1] = t.y;
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = wave_sum(v[k]);
  }
  if constexpr (WAVES > 1) {
    const int wv = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) s.buf[turn][wv][k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) t += s.buf[turn][i][k];
      v[k] = t;
    }
    turn ^= 1;
  }
}

template <int WAVES>
constexpr int kNormThreads = WAVES == 1 ? 256 : WAVES * kWave;
template <int WAVES>
constexpr int kNormRows = kNormThreads<WAVES> / (WAVES * kWave);  // rows of a workgroup at a time

// EIGHTS: C is a multiple of 8, so that no thread has a part of an eight: its selects and
// addresses cost registers (94 for 108 at 2048 16-bit channels, five waves a SIMD for
// four) and a test before each load. Forward of 16384 x 2048 bf16 26.5 with, 34 without;
// of 7 x 2048 f16 3.5 and 4.1, its gradient 4.5 and 5.5.
template <int FMT, int WFMT, int WAVES, int NC, bool EIGHTS>
__global__ __launch_bounds__(kNormThreads<WAVES>) void norm_kernel(NormArgs g) {
  __shared__ RowReduce<WAVES, 2> red;
  constexpr int T = WAVES * kWave;
  const int t = threadIdx.x % T, C = g.C;
  const float inv = 1.f / (float)C;
  int n[NC], turn = 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) n[c] = part_len(c * T + t, C);
#pragma unroll 1
  for (int64_t row = (int64_t)blockIdx.x * kNormRows<WAVES> + __builtin_amdgcn_readfirstlane(threadIdx.x / T); row < g.N;
       row += (int64_t)gridDim.x * kNormRows<WAVES>) {
    const char *src = static_cast<const char *>(g.x) + row * g.ldx * kLogitBytes<FMT>;
    char *dst = static_cast<char *>(g.y) + row * C * kLogitBytes<FMT>;
    Chunk<FMT> x[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) load_part<FMT, EIGHTS>(x[c], src, c * T + t, n[c]);
    auto diff = [&](int c, float s, float m, float (&d)[8]) {  // x s - m, 0 where there is no x
      x[c].get(d);
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = fmaf(d[e], s, -m);
      if (n[c] < 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (EIGHTS || e >= n[c]) d[e] = 0.f;
      }
    };
    float s, m, shift, var;
    auto stats = [&](float scale) {
      s = scale;
      float a[2] = {0.f, 0.f};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float d[8];
        diff(c, s, 0.f, d);
        a[0] += ((d[0] + d[1]) + (d[2] + d[3])) + ((d[4] + d[5]) + (d[6] + d[7]));
      }
      row_reduce(red, turn, a);
      m = a[0] * inv;
      // Where a sixteenth or less of the mean square about m is deviation (m is rounded: a few
      // steps of float32), once more about the corrected mean: else the variance is what
      // rounding leaves of m's error, 0 too, and the error comes out as a deviation.
#pragma unroll 1
      for (int turns = 0; turns < 2; ++turns) {
        // (one value: the compiler joins this product and some of the differences in an fma,
        // and two m of a row of one value are a deviation to an eps of 1e-12)
        asm volatile("" : "+v"(m));
        a[0] = a[1] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          float d[8];
          diff(c, s, m, d);
          a[0] += ((d[0] + d[1]) + (d[2] + d[3])) + ((d[4] + d[5]) + (d[6] + d[7]));
#pragma unroll
          for (int e = 0; e < 8; ++e) a[1] = fmaf(d[e], d[e], a[1]);
        }
        row_reduce(red, turn, a);
        shift = a[0] * inv;
        const float square = a[1] * inv;
        var = fmaxf(fmaf(-shift, shift, square), 0.f) + 0.f * a[1];  // (NaN and inf stay)
        if (turns > 0 || !(var < 0.0625f * square)) break;           // (the same for every lane of the row)
        m += shift;
      }
    };
    stats(1.f);
    if (!(var < 0x1p100f)) stats(kFarScale);  // (the same for every lane of the row)
    const double v = (double)var + g.eps * (double)s * (double)s;
    // (in 64 bits: of a row of one value that is taken times 2^-72, v is eps 2^-144 alone, which float32 has not)
    double r = __builtin_amdgcn_rsq(v);
    r = r * fma(-0.5 * v * r, r, 1.5);
    const float rs = (float)r;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float d[8], w[8], b[8];  // (from the CU's L1, which holds them: in registers they cost the row's own waves)
      load_part_f<WFMT, EIGHTS>(w, g.w, c * T + t, n[c]);
      load_part_f<WFMT, EIGHTS>(b, g.b, c * T + t, n[c]);
      diff(c, s, m, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = fmaf((d[e] - shift) * rs, w[e], b[e]);
      store_part<FMT, EIGHTS>(dst, c * T + t, n[c], d);
    }
    if (t == 0 && g.mean) {
      g.mean[row] = (m + shift) * (1.f / s);
      g.rstd[row] = (float)(r * (double)s);
    }
  }
}

template <int FMT, int WFMT, int WAVES, int NC, bool EIGHTS>
__global__ __launch_bounds__(kNormThreads<WAVES>) void norm_grad_kernel(NormGradArgs g) {
  __shared__ RowReduce<WAVES, 3> red;
  constexpr int T = WAVES * kWave, kRows = kNormRows<WAVES>;
  const int t = threadIdx.x % T, sub = __builtin_amdgcn_readfirstlane(threadIdx.x / T), C = g.C;
  const float inv = 1.f / (float)C;
  int n[NC], turn = 0;
  float w[NC][8], dw[NC][8], db[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    n[c] = part_len(c * T + t, C);
    load_part_f<WFMT, EIGHTS>(w[c], g.w, c * T + t, n[c]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[c][e] = db[c][e] = 0.f;
  }
  // the next row is on its way while one is worked on (but of 8 and 16 waves, which have no registers for it: 16 waves
  // have 128 each, and without it spill 19 of them in float32, and 2 in 16 bits where C is no multiple of 8)
  constexpr bool kAhead = WAVES <= 4;
  Chunk<FMT> xn[NC], yn[NC];
  float rstd_n, mean_n;
  auto fetch = [&](int64_t row) {
    const char *xs = static_cast<const char *>(g.x) + row * g.ldx * kLogitBytes<FMT>;
    const char *ys = static_cast<const char *>(g.dy) + row * g.lddy * kLogitBytes<FMT>;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      load_part<FMT, EIGHTS>(xn[c], xs, c * T + t, n[c]);
      load_part<FMT, EIGHTS>(yn[c], ys, c * T + t, n[c]);
    }
    rstd_n = g.rstd[row], mean_n = g.mean[row];
  };
  const int64_t step = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + sub;
  if (kAhead && row < g.N) fetch(row);
#pragma unroll 1
  for (; row < g.N; row += step) {
    if (!kAhead) fetch(row);
    char *dst = static_cast<char *>(g.dx) + row * C * kLogitBytes<FMT>;
    Chunk<FMT> x[NC], y[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) x[c] = xn[c], y[c] = yn[c];
    const float rstd = rstd_n, mean = mean_n;
    if (kAhead && row + step < g.N) fetch(row + step);
    const float s = rstd < 0x1p-50f ? kFarScale : 1.f, m = mean * s, rs = rstd * (1.f / s);
    float a[3] = {0.f, 0.f, 0.f};  // sums of g, g (x - m) and x - m
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float d[8], q[8];
      x[c].get(d);
      y[c].get(q);
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = fmaf(d[e], s, -m);
      if (n[c] < 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (EIGHTS || e >= n[c]) d[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float ge = q[e] * w[c][e];
        a[0] += ge;
        a[1] = fmaf(ge, d[e], a[1]);
        a[2] += d[e];
      }
    }
    row_reduce(red, turn, a);
    const float shift = a[2] * inv, c1 = a[0] * inv, c2 = rs * fmaf(-shift, a[0], a[1]) * inv;
#pragma unroll
    for (int c = 0; c < NC; ++c) x[c].opaque(), y[c].opaque();
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float d[8], q[8];
      x[c].get(d);
      y[c].get(q);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float xh = (fmaf(d[e], s, -m) - shift) * rs;
        dw[c][e] = fmaf(q[e], xh, dw[c][e]);
        db[c][e] += q[e];
        d[e] = rstd * fmaf(-xh, c2, fmaf(q[e], w[c][e], -c1));
      }
      store_part<FMT, EIGHTS>(dst, c * T + t, n[c], d);
    }
  }
  // the workgroup's sums: its waves' added by one wave a chunk
  float *part = g.part + (int64_t)blockIdx.x * 2 * C;
  if constexpr (kRows > 1) {
    static_assert(NC <= kRows);
    __shared__ float sum[2][kRows][NC * 8][T];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[0][sub][8 * c + e][t] = dw[c][e], sum[1][sub][8 * c + e][t] = db[c][e];
    __syncthreads();
    if (sub >= NC) return;
    const int len = part_len(sub * T + t, C);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = sum[k][0][8 * sub + e][t];
#pragma unroll
        for (int i = 1; i < kRows; ++i) v[e] += sum[k][i][8 * sub + e][t];
      }
      store_part<1, EIGHTS>(part + k * C, sub * T + t, len, v);
    }
  } else {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      store_part<1, EIGHTS>(part, c * T + t, n[c], dw[c]);
      store_part<1, EIGHTS>(part + C, c * T + t, n[c], db[c]);
    }
  }
}

// dw and db from the workgroups' sums [G][2 C]: 64 columns a workgroup, 16 waves on
// equal ranges of G, joined in 64 bits.
constexpr int kSumWaves = 16;
__global__ __launch_bounds__(kSumWaves *kWave) void norm_sum_kernel(const float *part, int G, int C, void *dw, void *db, int fmt) {
  __shared__ double s[kSumWaves][kWave];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, col = blockIdx.x * kWave + lane;
  const int per = (G + kSumWaves - 1) / kSumWaves, i0 = wv * per, i1 = min(G, i0 + per);
  double a = 0.0;
  if (col < 2 * C) {
#pragma unroll 8
    for (int i = i0; i < i1; ++i) a += (double)part[(int64_t)i * 2 * C + col];
  }
  s[wv][lane] = a;
  __syncthreads();
  if (wv != 0 || col >= 2 * C) return;
#pragma unroll
  for (int i = 1; i < kSumWaves; ++i) a += s[i][lane];
  void *out = col < C ? dw : db;
  const int at = col < C ? col : col - C;
  if (fmt == 1) static_cast<float *>(out)[at] = (float)a;
  else static_cast<uint16_t *>(out)[at] = f_to_u16((float)a, fmt == 2);
}

// Workgroups of the gradient: as many as a CU holds, their sums [2][C] each being written and read once more.
inline int64_t grad_blocks(int dtype, int64_t N, int C) {
  const int64_t n = C <= (dtype == 1 ? 1024 : 2048) ? (N + kNormRows<1> - 1) / kNormRows<1> : N, most = C <= 8192 ? 512 : 256;
  return n < most ? n : most;
}

// f(WAVES, NC, EIGHTS) for rows of C channels
template <int FMT, class F>
void with_shape(int C, F f) {
  using std::integral_constant;
#define RWKV7_SHAPE(W, N)                                                                   \
  C % 8 == 0 ? f(integral_constant<int, W>(), integral_constant<int, N>(), std::true_type()) \
             : f(integral_constant<int, W>(), integral_constant<int, N>(), std::false_type())
  if (C <= 512) RWKV7_SHAPE(1, 1);
  else if (C <= 1024) RWKV7_SHAPE(1, 2);
  else if (C <= 2048) {
    if constexpr (FMT == 1) RWKV7_SHAPE(4, 1);
    else RWKV7_SHAPE(1, 4);
  } else if (C <= 4096) RWKV7_SHAPE(4, 2);
  else if (C <= 8192) RWKV7_SHAPE(8, 2);
  else RWKV7_SHAPE(16, 2);
#undef RWKV7_SHAPE
}

// f(FMT, WFMT) for the two types
template <class F>
void with_types(int dtype, int wtype, F f) {
  using std::integral_constant;
  using F16 = integral_constant<int, 0>;
  using F32 = integral_constant<int, 1>;
  using BF16 = integral_constant<int, 2>;
  if (dtype == 1) f(F32(), F32());
  else if (dtype == 0) wtype == 1 ? f(F16(), F32()) : f(F16(), F16());
  else wtype == 1 ? f(BF16(), F32()) : f(BF16(), BF16());
}

bool types_ok(int dtype, int wtype) { return dtype >= 0 && dtype <= 2 && (wtype == 1 || wtype == dtype); }

}  // namespace
}  // namespace rwkv7

extern "C" int rwkv7_layer_norm_forward(const void *x, int32_t dtype, int64_t ldx, const void *weight, const void *bias,
                                        int32_t weight_dtype, double eps, void *y, float *mean, float *rstd, int64_t N,
                                        int32_t C, void *stream) {
  using namespace rwkv7;
  if (!x || !weight || !bias || !y || !mean != !rstd || !types_ok(dtype, weight_dtype)) return RWKV7_EINVAL;
  if (!(eps >= 1e-30 && eps <= 1e30)) return RWKV7_EINVAL;
  if (N < 1 || C < 1 || C > kNormMaxC || ldx < C) return RWKV7_ESHAPE;
  const NormArgs g = {x, weight, bias, ldx, y, mean, rstd, N, C, eps};
  with_types(dtype, weight_dtype, [&](auto f, auto wf) {
    with_shape<decltype(f)::value>(C, [&](auto waves, auto nc, auto eights) {
      constexpr int W = decltype(waves)::value;
      const int64_t n = (N + kNormRows<W> - 1) / kNormRows<W>;
      norm_kernel<decltype(f)::value, decltype(wf)::value, W, decltype(nc)::value, decltype(eights)::value>
          <<<(int)(n < (1 << 20) ? n : 1 << 20), kNormThreads<W>, 0, static_cast<hipStream_t>(stream)>>>(g);
    });
  });
  RWKV7_CHECK_LAUNCH();
  return RWKV7_OK;
}

extern "C" int64_t rwkv7_layer_norm_backward_workspace_bytes(int32_t dtype, int64_t N, int32_t C) {
  using namespace rwkv7;
  if (N < 1 || C < 1 || C > kNormMaxC) return 0;
  return grad_blocks(dtype, N, C) * 2 * C * 4;
}

extern "C" int rwkv7_layer_norm_backward(const void *grad_y, int64_t ldg, const void *x, int64_t ldx, int32_t dtype,
                                         const void *weight, int32_t weight_dtype, const float *mean, const float *rstd,
                                         void *grad_x, void *grad_weight, void *grad_bias, int64_t N, int32_t C,
                                         void *workspace, int64_t workspace_bytes, void *stream) {
  using namespace rwkv7;
  if (!grad_y || !x || !weight || !mean || !rstd || !grad_x || !grad_weight || !grad_bias || !workspace) return RWKV7_EINVAL;
  if (!types_ok(dtype, weight_dtype)) return RWKV7_EINVAL;
  if (N < 1 || C < 1 || C > kNormMaxC || ldx < C || ldg < C) return RWKV7_ESHAPE;
  if (workspace_bytes < rwkv7_layer_norm_backward_workspace_bytes(dtype, N, C)) return RWKV7_EWORKSPACE;
  float *part = static_cast<float *>(workspace);
  const NormGradArgs g = {grad_y, x, weight, ldg, ldx, mean, rstd, grad_x, part, N, C};
  const int G = (int)grad_blocks(dtype, N, C);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  with_types(dtype, weight_dtype, [&](auto f, auto wf) {
    with_shape<decltype(f)::value>(C, [&](auto waves, auto nc, auto eights) {
      constexpr int W = decltype(waves)::value;
      norm_grad_kernel<decltype(f)::value, decltype(wf)::value, W, decltype(nc)::value, decltype(eights)::value>
          <<<G, kNormThreads<W>, 0, st>>>(g);
    });
  });
  RWKV7_CHECK_LAUNCH();
  norm_sum_kernel<<<(2 * C + kWave - 1) / kWave, kSumWaves * kWave, 0, st>>>(part, G, C, grad_weight, grad_bias, weight_dtype);
  RWKV7_CHECK_LAUNCH();
  return RWKV7_OK;
}
