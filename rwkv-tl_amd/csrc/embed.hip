// Embedding lookup with a factor, and the table's gradient.
//
//   out[i, :] = s W[t_i, :]               zeros where t_i is outside 0 .. V-1
//   dW[v, :]  = s sum_{i: t_i = v} dy[i, :]     zeros where there is none
// The sums are in 32 bits, each token's rows added up in an order that the tokens
// alone decide: the same call gives the same bits.
//
// Gradient. The table's rows belong to G workgroups, row v to workgroup v % G (frequent
// tokens have neighbouring ids). Each counts the tokens of its rows, and reads the
// tokens once more for their positions. Rows of up to 64 positions are summed by a wave
// each, their positions brought into order first by counting; rows without any are
// written as zeros by the waves that are free. The positions of a row with more go, in
// order, to a list in the workspace, in units of about 64 that a second launch sums,
// four waves a unit; the unit that arrives last at its row adds up the units' sums.
//
// Bound by the table's own bytes, written once; nothing is cleared first.
#include "row_parts.h"
#include "rwkv7_kernels.h"

namespace rwkv7 {
namespace {

constexpr int64_t kEmbedMaxN = (1 << 26) - 4;  // (a grid has fewer than 2^32 threads)
constexpr int kEmbedMaxV = 1 << 20, kEmbedMaxC = 65536;

struct EmbedArgs {
  const void *w;
  int64_t ldw;
  const int64_t *tokens;
  void *out;
  int64_t N;
  int V, C;
  float scale;
};

// A wave per row and 64 eights of it.
template <int FMT>
__global__ __launch_bounds__(256) void embed_kernel(EmbedArgs g) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= g.N) return;
  const int64_t id = g.tokens[row];
  const bool there = id >= 0 && id < g.V;
  const char *src = static_cast<const char *>(g.w) + (there ? id : 0) * g.ldw * kLogitBytes<FMT>;
  char *dst = static_cast<char *>(g.out) + row * g.C * kLogitBytes<FMT>;
#pragma unroll 4
  for (int b = lane; b < (g.C + 7) / 8; b += kWave) {
    const int n = part_len(b, g.C);
    float f[8] = {};
    if (there) {
      load_part_f<FMT>(f, src, b, n);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= g.scale;
    }
    store_part<FMT>(dst, b, n, f);
  }
}

// ---- gradient -----------------------------------------------------------------

constexpr int kOwnThreads = 1024, kOwnWaves = kOwnThreads / kWave;
constexpr int kOwnRows = 256;  // rows of a workgroup at most
constexpr int kFew = 64;       // positions that a wave sums by itself
constexpr int kUnit = 64;      // positions of a unit of a longer row, while these make no more than
constexpr int kMaxUnits = 256; // units a row
constexpr int kCols = 512;     // columns of a unit's workgroup

struct Unit {
  int row;           // -1: none
  int start, count;  // of the list of positions
  int first, units;  // the row's first unit and how many it has
};

struct EmbedGradArgs {
  const void *dy;
  int64_t ldg;
  const int64_t *tokens;
  void *out;
  int64_t N;
  int V, C, log_g;
  float scale;
  // for N > kFew
  int *order;    // [N]
  Unit *table;   // [slots]
  int *arrived;  // [slots][column blocks]
  float *part;   // [slots][C]
  int slots, blocks;
};

struct OwnLds {
  int count[kOwnRows];
  int at[kOwnRows];       // of a row of few: where its next position goes
  int few[kOwnRows];      // rows of 1 .. kFew positions, then (from the end) those of none
  int hot[kOwnRows];      // rows of more
  int n_few, n_none, n_hot, next, less;
  int wave[kOwnWaves];
  uint32_t list[kOwnRows * kFew];
};

// Exclusive sum over the first kOwnRows threads (four waves) of the workgroup.
RWKV7_DEV int own_scan(int v, int *wave, int &total) {
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  int inc = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int o = __shfl_up(inc, d);
    if (lane >= d) inc += o;
  }
  __syncthreads();
  if (lane == kWave - 1) wave[wv] = inc;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kOwnRows / kWave; ++i) {
    before += i < wv ? wave[i] : 0;
    total += wave[i];
  }
  return before + inc - v;
}

template <int FMT>
RWKV7_DEV void add_eight(float (&acc)[8], const Chunk<FMT> &x) {
  float f[8];
  x.get(f);
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] += f[e];
}

template <int FMT>
__global__ __launch_bounds__(kOwnThreads) void embed_grad_kernel(EmbedGradArgs a) {
  __shared__ OwnLds s;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, g = blockIdx.x, G = 1 << a.log_g;
  const int rows = g < a.V ? ((a.V - 1 - g) >> a.log_g) + 1 : 0;  // <= kOwnRows
  if (t < kOwnRows) s.count[t] = 0;
  if (t == 0) s.n_few = s.n_none = s.n_hot = s.next = s.less = 0;
  __syncthreads();

  // how often each row's token occurs, and how many tokens belong to workgroups before
  int less = 0;
#pragma unroll 4
  for (int64_t i = t; i < a.N; i += kOwnThreads) {
    const int64_t id = a.tokens[i];
    if (id >= 0 && id < a.V) {
      const int owner = (int)id & (G - 1);
      if (owner == g) atomicAdd(&s.count[(int)id >> a.log_g], 1);
      less += owner < g;
    }
  }
  if (a.slots) {
    less = (int)(wave_sum_d((double)less));
    if (lane == 0) atomicAdd(&s.less, less);
  }
  __syncthreads();
  const int c = t < rows ? s.count[t] : 0;
  int few_total, all;
  const int few_at = own_scan(c <= kFew ? c : 0, s.wave, few_total);
  const int all_at = own_scan(c, s.wave, all);
  if (t < rows) {
    s.at[t] = few_at;
    if (c == 0) s.few[kOwnRows - 1 - atomicAdd(&s.n_none, 1)] = t;
    else if (c <= kFew) s.few[atomicAdd(&s.n_few, 1)] = t;
    else s.hot[atomicAdd(&s.n_hot, 1)] = t;
  }
  __syncthreads();

  // the rows of few positions: these in any order, sorted below
#pragma unroll 4
  for (int64_t i = t; i < a.N; i += kOwnThreads) {
    const int64_t id = a.tokens[i];
    if (id >= 0 && id < a.V && ((int)id & (G - 1)) == g) {
      const int r = (int)id >> a.log_g;
      if (s.count[r] <= kFew) s.list[atomicAdd(&s.at[r], 1)] = (uint32_t)i;
    }
  }

  // the units of the others. A workgroup's tokens are its range of the list; a row of c
  // has no more than c / 32 units, so that its units have a range of the table likewise.
  if (a.slots) {
    const int base = s.less, slot0 = (base + 31) / 32;
    int slot1 = (base + all + 31) / 32;
    if (g == G - 1) slot1 = a.slots;
    const bool hot = t < rows && c > kFew;
    const int units = hot ? min((c + kUnit - 1) / kUnit, kMaxUnits) : 0, per = hot ? (c + units - 1) / units : 0;
    int used;
    const int first = own_scan(units, s.wave, used) + slot0;
    for (int u = 0; u < units; ++u) {
      const int from = min(u * per, c), to = min(from + per, c);
      a.table[first + u] = {(t << a.log_g) + g, base + all_at + from, to - from, first, units};
    }
    for (int i = slot0 + used + t; i < slot1; i += kOwnThreads) a.table[i].row = -1;
    for (int64_t i = (int64_t)slot0 * a.blocks + t; i < (int64_t)(slot0 + used) * a.blocks; i += kOwnThreads) a.arrived[i] = 0;
    // their positions in order: each wave a range of the tokens, first counted
    if (t < rows) s.at[t] = c > kFew ? base + all_at : s.at[t];
    __syncthreads();
    const int64_t span = ((a.N + kOwnWaves - 1) / kOwnWaves + kWave - 1) / kWave * kWave;
    const int64_t i0 = wv * span, i1 = min(a.N, i0 + span);
    for (int h = 0; h < s.n_hot; ++h) {
      const int r = s.hot[h];
      const int64_t want = ((int64_t)r << a.log_g) + g;
      int n = 0;
#pragma unroll 4
      for (int64_t i = i0; i < i1; i += kWave) n += __popcll(__ballot(i + lane < i1 && a.tokens[min(i + lane, a.N - 1)] == want));
      __syncthreads();
      if (lane == 0) s.wave[wv] = n;
      __syncthreads();
      int at = s.at[r];
      for (int i = 0; i < wv; ++i) at += s.wave[i];
      if (n > 0) {
#pragma unroll 4
        for (int64_t i = i0; i < i1; i += kWave) {
          const bool is = i + lane < i1 && a.tokens[min(i + lane, a.N - 1)] == want;
          const u64 m = __ballot(is);
          if (is) a.order[at + __popcll(m & ((1ull << lane) - 1))] = (int)(i + lane);
          at += __popcll(m);
        }
      }
    }
  }
  __syncthreads();

  // a row at a time, to whichever wave is free: first those with positions
  const int n_few = s.n_few, n_rows = n_few + s.n_none, n8 = (a.C + 7) / 8;
  for (;;) {
    int k = lane == 0 ? atomicAdd(&s.next, 1) : 0;
    k = __builtin_amdgcn_readfirstlane(k);
    if (k >= n_rows) break;
    const int r = s.few[k < n_few ? k : kOwnRows - 1 - (k - n_few)];
    char *dst = static_cast<char *>(a.out) + (((int64_t)r << a.log_g) + g) * a.C * kLogitBytes<FMT>;
    if (k >= n_few) {
      const float zero[8] = {};
      for (int b = lane; b < n8; b += kWave) store_part<FMT>(dst, b, part_len(b, a.C), zero);
      continue;
    }
    const int n = __builtin_amdgcn_readfirstlane(s.count[r]), at = __builtin_amdgcn_readfirstlane(s.at[r]) - n;
    uint32_t pos = lane < n ? s.list[at + lane] : ~0u;
    if (n > 1) {
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += (uint32_t)__builtin_amdgcn_readlane((int)pos, j) < pos;
      if (lane < n) s.list[at + rank] = pos;
      __builtin_amdgcn_wave_barrier();
      pos = lane < n ? s.list[at + lane] : 0u;
    }
    for (int b = lane; b < (n8 + kWave - 1) / kWave * kWave; b += kWave) {
      const int len = part_len(b, a.C);
      float acc[8] = {};
#pragma unroll 8
      for (int j = 0; j < n; ++j) {
        const uint32_t p = (uint32_t)__builtin_amdgcn_readlane((int)pos, j);
        Chunk<FMT> x;
        load_part(x, static_cast<const char *>(a.dy) + p * a.ldg * kLogitBytes<FMT>, b, len);
        add_eight(acc, x);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] *= a.scale;
      store_part<FMT>(dst, b, len, acc);
    }
  }
}

// A unit's 512 columns: wave w sums the positions w, w + 4, ..; the waves' sums, and the
// units', are added in order.
template <int FMT>
__global__ __launch_bounds__(256) void embed_unit_kernel(EmbedGradArgs a) {
  __shared__ float sum[4][kCols];
  __shared__ bool last;
  const Unit u = a.table[blockIdx.x];
  if (u.row < 0) return;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, b = blockIdx.y * (kCols / 8) + lane, len = part_len(b, a.C);
  float acc[8] = {};
  if (len > 0) {
#pragma unroll 8
    for (int j = wv; j < u.count; j += 4) {
      const int64_t p = a.order[u.start + j];
      Chunk<FMT> x;
      load_part(x, static_cast<const char *>(a.dy) + p * a.ldg * kLogitBytes<FMT>, b, len);
      add_eight(acc, x);
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[wv][8 * lane + e] = acc[e];
  __syncthreads();
  const int64_t col0 = (int64_t)blockIdx.y * kCols + 2 * t;
  float v[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    v[e] = (sum[0][2 * t + e] + sum[1][2 * t + e]) + (sum[2][2 * t + e] + sum[3][2 * t + e]);
    // stored past the caches of this XCD, acknowledged before the count goes up
    if (col0 + e < a.C)
      __hip_atomic_store(a.part + (int64_t)blockIdx.x * a.C + col0 + e, v[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (t == 0)
    last = __hip_atomic_fetch_add(a.arrived + (int64_t)u.first * a.blocks + blockIdx.y, 1, __ATOMIC_RELAXED,
                                  __HIP_MEMORY_SCOPE_AGENT) == u.units - 1;
  __syncthreads();
  if (!last) return;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (col0 + e >= a.C) break;
    const float *p = a.part + (int64_t)u.first * a.C + col0 + e;
    float total = 0.f;
#pragma unroll 8
    for (int i = 0; i < u.units; ++i)
      total += __hip_atomic_load(p + (int64_t)i * a.C, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    store_logit<FMT>(a.out, u.row * (int64_t)a.C + col0 + e, total * a.scale);
  }
}

int log_groups(int V) {
  int l = 8;
  while ((int64_t)kOwnRows << l < V) ++l;
  return l;
}

struct GradSpace {
  int64_t table, arrived, order, part, bytes;
  int slots, blocks;
};
GradSpace grad_space(int64_t N, int C) {
  GradSpace s = {};
  if (N <= kFew) return s;  // no row has more
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  s.slots = (int)((N + 31) / 32);
  s.blocks = (C + kCols - 1) / kCols;
  s.table = 0;
  s.arrived = s.table + up(s.slots * (int64_t)sizeof(Unit));
  s.order = s.arrived + up((int64_t)s.slots * s.blocks * 4);
  s.part = s.order + up(N * 4);
  s.bytes = s.part + (int64_t)s.slots * C * 4;
  return s;
}

bool sizes_ok(int64_t N, int V, int C) {
  return N >= 1 && N <= kEmbedMaxN && V >= 1 && V <= kEmbedMaxV && C >= 1 && C <= kEmbedMaxC;
}

}  // namespace
}  // namespace rwkv7

extern "C" int rwkv7_embed(const void *weight, int32_t dtype, int64_t ldw, const int64_t *tokens, float scale, void *out,
                           int64_t N, int32_t V, int32_t C, void *stream) {
  using namespace rwkv7;
  if (!weight || !tokens || !out || dtype < 0 || dtype > 2) return RWKV7_EINVAL;
  if (!sizes_ok(N, V, C) || ldw < C) return RWKV7_ESHAPE;
  const EmbedArgs g = {weight, ldw, tokens, out, N, V, C, scale};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int grid = (int)((N + 3) / 4);
  switch (dtype) {
    case 0: embed_kernel<0><<<grid, 256, 0, st>>>(g); break;
    case 1: embed_kernel<1><<<grid, 256, 0, st>>>(g); break;
    default: embed_kernel<2><<<grid, 256, 0, st>>>(g); break;
  }
  RWKV7_CHECK_LAUNCH();
  return RWKV7_OK;
}

extern "C" int64_t rwkv7_embed_backward_workspace_bytes(int64_t N, int32_t V, int32_t C) {
  using namespace rwkv7;
  return sizes_ok(N, V, C) ? grad_space(N, C).bytes : 0;
}

extern "C" int rwkv7_embed_backward(const void *grad, int32_t dtype, int64_t ldg, const int64_t *tokens, float scale,
                                    void *grad_weight, int64_t N, int32_t V, int32_t C, void *workspace,
                                    int64_t workspace_bytes, void *stream) {
  using namespace rwkv7;
  if (!grad || !tokens || !grad_weight || dtype < 0 || dtype > 2) return RWKV7_EINVAL;
  if (!sizes_ok(N, V, C) || ldg < C) return RWKV7_ESHAPE;
  const GradSpace s = grad_space(N, C);
  if (s.bytes && !workspace) return RWKV7_EINVAL;
  if (workspace_bytes < s.bytes) return RWKV7_EWORKSPACE;
  char *ws = static_cast<char *>(workspace);
  const int l = log_groups(V);
  const EmbedGradArgs a = {grad, ldg, tokens, grad_weight, N, V, C, l, scale, reinterpret_cast<int *>(ws + s.order),
                           reinterpret_cast<Unit *>(ws + s.table), reinterpret_cast<int *>(ws + s.arrived),
                           reinterpret_cast<float *>(ws + s.part), s.slots, s.blocks};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case 0: embed_grad_kernel<0><<<1 << l, kOwnThreads, 0, st>>>(a); break;
    case 1: embed_grad_kernel<1><<<1 << l, kOwnThreads, 0, st>>>(a); break;
    default: embed_grad_kernel<2><<<1 << l, kOwnThreads, 0, st>>>(a); break;
  }
  RWKV7_CHECK_LAUNCH();
  if (s.slots) {
    const dim3 grid(s.slots, s.blocks);
    switch (dtype) {
      case 0: embed_unit_kernel<0><<<grid, 256, 0, st>>>(a); break;
      case 1: embed_unit_kernel<1><<<grid, 256, 0, st>>>(a); break;
      default: embed_unit_kernel<2><<<grid, 256, 0, st>>>(a); break;
    }
    RWKV7_CHECK_LAUNCH();
  }
  return RWKV7_OK;
}
