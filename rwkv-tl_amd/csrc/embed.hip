// Embedding lookup with a factor, and the table's gradient.
//
//   out[i, :] = s W[t_i, :]               zeros where t_i is outside 0 .. V-1
//   dW[v, :]  = s sum_{i: t_i = v} dy[i, :]     zeros where there is none
// The sums are in 32 bits, each token's rows added up in an order that the tokens
// alone decide: the same call gives the same bits.
//
// Gradient, two launches. The first sorts the positions by token, and beside that fills
// the table with zeros: V C values, most of what the call has to move, which hide the
// sort's latency (the rows that the second launch writes are so written twice: one in
// twelve of 65536 for 16384 tokens).
//   Sort: the table's rows belong to G workgroups, row v to workgroup v % G (frequent
//   tokens have neighbouring ids). Each counts the tokens of its rows and those of the
//   workgroups before it, which gives its range of the list of positions, and reads the
//   tokens once more for the positions. Those of a row of up to 64 are put in order by
//   counting the lesser ones. Of rows with more, the second pass counts each wave's share
//   and a third, if there is such a row, meets the positions in order: three passes
//   however many there are (with two for each, 2^20 tokens of 8192 ids took 26 ms, 2^22 of
//   65536 461; now 1.15 and 5.0).
// The second launch goes through the sorted list, eight positions a workgroup and what
// else belongs to the rows that begin there, so that eight rows are always in flight. A
// row of more than 32 positions is cut into units; the one that arrives last adds up
// the units' sums.
//
// Measured (kernel trace, us; tokens with frequencies of 1 / rank; a large copy moves 5.09
// TB/s here, a large fill 6.9-7.9). 8192 tokens x 1024 of 65536 bf16: sort and fill 20
// (6.7 TB/s), sums 11; 16384 x 2048: 40 and 36, the second beside the first's lines on their
// way from the caches; 509 x 768 of 20011 f32: 12 and 5. Sort alone 6.7 for one token, 14
// for 16384; past those that its threads hold (16384) it reads them again, about 1 for every
// 1024 (65536: 57, 2^20: 1080, and 685 with no row of more than 64). 16384 x 2048 of one
// id: 45-51 and 120 (128 units of 128 positions, on half of the CUs), half of them one id 47
// and 54. Lookup of 16384 x 2048 bf16 28 (4.8 TB/s), of the same ids again 17, f32 36; of 16
// 2.8. Tried: a wave a row in the sort's workgroups, zeros and sums
// included (the table's rows of 16384 x 2048: 179; the longest rows' chains bound it);
// units of 64 positions (sums of 8192 x 1024 10.0 -> 11.9); the sums of a unit stored 32
// bytes a thread (27 instead of 10: each 4-byte store past the caches is a trip of its own).
#include "logits_rows.h"
#include "rwkv7_kernels.h"

namespace rwkv7 {
namespace {

constexpr int64_t kEmbedMaxN = (1 << 24) - 1;  // (a grid has fewer than 2^32 threads)
constexpr int kEmbedMaxV = 1 << 20, kEmbedMaxC = 65536;

// A thread's piece of a row: E values, 16 bytes or (rows shorter than that) one value. The
// last piece of a row ends with it, over the one before where E does not divide C: both
// have the same values there. Rows may start at any element.
template <int FMT, int E>
RWKV7_DEV int piece_at(int b, int C) {
  return min(E * b, C - E);
}
template <int FMT, int E>
struct Piece {
  uint32_t w[E == 1 ? 1 : 4];
  RWKV7_DEV void load(const char *p) {
    if constexpr (E > 1) __builtin_memcpy(w, p, 16);
    else if constexpr (FMT == 1) w[0] = *reinterpret_cast<const uint32_t *>(p);
    else w[0] = *reinterpret_cast<const uint16_t *>(p);
  }
  RWKV7_DEV void get(float (&f)[E]) const {
    if constexpr (FMT == 1) {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = __uint_as_float(w[e]);
    } else if constexpr (E == 1) {
      f[0] = F16T<FMT == 2>::to_f((uint16_t)w[0]);
    } else {
      F16T<FMT == 2>::to_f8(make_uint4(w[0], w[1], w[2], w[3]), f);
    }
  }
};
template <int FMT, int E>
RWKV7_DEV void store_piece(char *p, const float (&f)[E]) {
  if constexpr (E == 1) {
    store_logit<FMT>(p, 0, f[0]);
  } else if constexpr (FMT == 1) {
    __builtin_memcpy(p, f, 16);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (uint32_t)F16T<FMT == 2>::from_f(f[2 * i]) | ((uint32_t)F16T<FMT == 2>::from_f(f[2 * i + 1]) << 16);
    __builtin_memcpy(p, w, 16);
  }
}
template <int FMT>
constexpr int kWide = FMT == 1 ? 4 : 8;
template <int E>
int pieces(int C) {
  return (C + E - 1) / E;
}

struct EmbedArgs {
  const void *w;
  int64_t ldw;
  const int64_t *tokens;
  void *out;
  int64_t N;
  int V, C;
  float scale;
};

// A wave per row.
template <int FMT, int E>
__global__ __launch_bounds__(256) void embed_kernel(EmbedArgs g) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= g.N) return;
  const int64_t id = g.tokens[row];
  const bool there = id >= 0 && id < g.V;
  const char *src = static_cast<const char *>(g.w) + (there ? id : 0) * g.ldw * kLogitBytes<FMT>;
  char *dst = static_cast<char *>(g.out) + row * g.C * kLogitBytes<FMT>;
#pragma unroll 4
  for (int b = lane; E * b < g.C; b += kWave) {
    const int at = piece_at<FMT, E>(b, g.C) * kLogitBytes<FMT>;
    float f[E] = {};
    if (there) {
      Piece<FMT, E> x;
      x.load(src + at);
      x.get(f);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] *= g.scale;
    }
    store_piece<FMT, E>(dst + at, f);
  }
}

// ---- gradient -----------------------------------------------------------------

constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kSortRows = 256;   // rows of a workgroup at most (8 bits beside a position's 24)
constexpr int kFew = 64;         // positions of a row that are ordered by counting
constexpr int kUnit = 32;        // positions of a unit at most, while a row has no more units than
constexpr int kMaxUnits = 128;
constexpr int kRun = 8;          // positions of the list, and rows in flight, of a workgroup
constexpr int kJoin = 4;         // units' sums in flight
constexpr int kFillGroups = 1024, kFillBytes = 1 << 16;  // workgroups of the fill at most, and bytes of each at least
constexpr int kHeld = 16;        // tokens that a thread of the sort keeps, where there are no more

// What begins at a position of the list.
struct Unit {
  int row;    // -1: nothing does
  int count;  // positions
  int at;     // which of its row's units this is, and 2^16 times how many it has
  int slot;   // of the row's first unit
};

struct EmbedGradArgs {
  const void *dy;
  int64_t ldg;
  const int64_t *tokens;
  void *out;
  int64_t N;
  int V, C, log_g;
  float scale;
  int *order;    // [N]
  Unit *table;   // [N]
  int *arrived;  // [slots][column blocks]: units that have arrived, at a row's first slot
  float *part;   // [slots][columns, whole workgroups]: sums of the units of rows that have several
  int blocks;
};

// A row of several units (33 positions or more) has a slot for each, behind those of the rows before it: no more
// than one for every 16 positions.
RWKV7_DEV int first_slot(int start) { return (start + 15) / 16; }
inline int64_t slots(int64_t N) { return (N + 15) / 16; }

// A row of c > kUnit positions has units_of(c) units of c / units, rounded down or up: 16 at
// least, so that behind one that begins among a workgroup's eight no other does.
RWKV7_DEV int units_of(int c) { return min((c + kUnit - 1) / kUnit, kMaxUnits); }
RWKV7_DEV int unit_start(int c, int units, int unit) { return (int)((uint32_t)unit * (uint32_t)c / (uint32_t)units); }
static_assert((uint64_t)kMaxUnits * kEmbedMaxN < 1ull << 32);

struct SortLds {
  int count[kSortRows];
  int at[kSortRows];    // of a row's positions in the list
  int few[kSortRows];   // of a row of few: in `keys`
  int next[kSortRows];  // where its next one goes there; of a row of more its counters there
  int hot[kSortRows];   // rows of more than kFew
  int n_hot, less;
  int wave[kSortWaves];
  // Row and position of those of rows of few; and behind them, a word left out, for each row of
  // more a counter of each wave (16 words for the 64 that the row has not taken).
  uint32_t keys[kSortRows * kFew];
  static_assert(kSortWaves < kFew);
};

// Exclusive sum over the first kSortRows threads (four waves) of the workgroup.
RWKV7_DEV int sort_scan(int v, int *wave, int &total) {
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
  for (int i = 0; i < kSortRows / kWave; ++i) {
    before += i < wv ? wave[i] : 0;
    total += wave[i];
  }
  return before + inc - v;
}

RWKV7_DEV void fill_zeros(char *out, int64_t bytes, int group, int groups) {
  const int64_t n16 = bytes / 16, step = (int64_t)groups * kSortThreads;
  const uint32_t zero[4] = {0u, 0u, 0u, 0u};
#pragma unroll 4
  for (int64_t i = (int64_t)group * kSortThreads + threadIdx.x; i < n16; i += step) __builtin_memcpy(out + 16 * i, zero, 16);
  if (group == 0 && threadIdx.x < bytes % 16) out[16 * n16 + threadIdx.x] = 0;
}

// HELD: each thread has its tokens in registers after the first pass. (Each trip to memory beside the fill's
// stores takes 2 us or more.)
template <int ELEM, bool HELD>
__global__ __launch_bounds__(kSortThreads, 8) void embed_sort_kernel(EmbedGradArgs a) {
  __shared__ SortLds s;
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6, g = blockIdx.x, G = 1 << a.log_g;
  if (g >= G) {
    fill_zeros(static_cast<char *>(a.out), (int64_t)a.V * a.C * ELEM, g - G, gridDim.x - G);
    return;
  }
  const int rows = g < a.V ? ((a.V - 1 - g) >> a.log_g) + 1 : 0;  // <= kSortRows
  if (t < kSortRows) s.count[t] = 0;
  if (t == 0) s.n_hot = s.less = 0;
  __syncthreads();

  // Wave w has the w-th range of the tokens, 64 at a time: f(position, the token's row
  // here or -1) for each.
  const int N = (int)a.N, span = ((N + kSortWaves - 1) / kSortWaves + kWave - 1) / kWave * kWave;
  const int i0 = wv * span, i1 = min(N, i0 + span);
  auto row_of = [&](int64_t id) { return id >= 0 && id < a.V && ((int)id & (G - 1)) == g ? (int)id >> a.log_g : -1; };
  int held[HELD ? kHeld : 1];
  auto each = [&](auto f) {
    if constexpr (HELD) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        if (i0 + k * kWave < i1) f(i0 + k * kWave + lane, held[k]);
    } else {
#pragma unroll 4
      for (int i = i0; i < i1; i += kWave) f(i + lane, i + lane < i1 ? row_of(a.tokens[i + lane]) : -1);
    }
  };

  // how often each row's token occurs, and how many tokens belong to workgroups before
  int less = 0;
  auto count = [&](int64_t id) {
    const int r = row_of(id);
    if (r >= 0) atomicAdd(&s.count[r], 1);
    less += id >= 0 && id < a.V && ((int)id & (G - 1)) < g;
    return r;
  };
  if constexpr (HELD) {
#pragma unroll
    for (int k0 = 0; k0 < kHeld; k0 += 8) {
      int64_t id[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int i = i0 + (k0 + k) * kWave + lane;
        id[k] = i < i1 ? a.tokens[i] : -1;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) held[k0 + k] = count(id[k]);
    }
  } else {
#pragma unroll 8
    for (int i = i0 + lane; i < i1; i += kWave) count(a.tokens[i]);
  }
  less = (int)wave_sum_d((double)less);
  if (lane == 0) atomicAdd(&s.less, less);
  __syncthreads();
  const int c = t < rows ? s.count[t] : 0;
  int all, n_few;
  const int at = sort_scan(c, s.wave, all) + s.less;
  const int few = sort_scan(c <= kFew ? c : 0, s.wave, n_few);
  if (t < rows) s.at[t] = at, s.few[t] = s.next[t] = few;
  if (c > kFew) {
    const int h = atomicAdd(&s.n_hot, 1);
    s.hot[h] = t;
    s.next[t] = n_few + 1 + h * kSortWaves;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) s.keys[s.next[t] + w] = 0u;
  }
  if (c > kUnit)
    for (int b = 0; b < a.blocks; ++b) a.arrived[(int64_t)first_slot(at) * a.blocks + b] = 0;
  if (g == G - 1)
    for (int i = s.less + all + t; i < N; i += kSortThreads) a.table[i].row = -1;
  __syncthreads();

  each([&](int i, int r) {
    if (r < 0) return;
    if (s.count[r] <= kFew) s.keys[atomicAdd(&s.next[r], 1)] = ((uint32_t)r << 24) | (uint32_t)i;
    else atomicAdd(&s.keys[s.next[r] + wv], 1u);
  });
  __syncthreads();
  for (int i = t; i < n_few; i += kSortThreads) {
    const uint32_t key = s.keys[i];
    const int r = key >> 24, from = s.few[r], n = s.count[r], start = s.at[r];
    int rank = 0;
    for (int j = from; j < from + n; ++j) rank += s.keys[j] < key;
    const int units = n > kUnit ? 2 : 1, per = n / units;  // (no more: kFew is two units)
    Unit u = {-1, 0, 0, 0};
    if (rank == 0 || rank == per) u = {(r << a.log_g) + g, rank == 0 ? per : n - per, (rank != 0) | (units << 16), first_slot(start)};
    a.order[start + rank] = (int)(key & 0xffffffu);
    a.table[start + rank] = u;
  }
  if (s.n_hot == 0) return;
  // rows of more, all in one pass: each wave's place in the list for each, and from there
  // its range of the tokens in order
  if (t < s.n_hot) {
    const int r = s.hot[t];
    uint32_t *const to = s.keys + s.next[r];
    uint32_t place = (uint32_t)s.at[r];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t n = to[w];
      to[w] = place;
      place += n;
    }
  }
  __syncthreads();
  each([&](int i, int r) {
    const int of = r >= 0 ? s.next[r] : 0;  // (no row of few has come further than n_few)
    u64 left = __ballot(of > n_few);
    while (left) {  // a row of the 64 tokens' a turn
      const int row = __builtin_amdgcn_readlane(of, __builtin_ctzll(left));
      const u64 m = __ballot(of == row);
      const uint32_t first = s.keys[row + wv];
      if (of == row) {
        const uint32_t place = first + __popcll(m & ((1ull << lane) - 1));
        a.order[place] = i;
        a.table[place].row = -1;
      }
      s.keys[row + wv] = first + __popcll(m);  // (by every lane, so that each reads what it wrote)
      left &= ~m;
    }
  });
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();  // the units' entries come after the positions' own
  for (int i = t; i < s.n_hot * kMaxUnits; i += kSortThreads) {
    const int r = s.hot[i / kMaxUnits], unit = i % kMaxUnits, total = s.count[r], start = s.at[r], units = units_of(total);
    if (unit >= units) continue;
    const int begin = unit_start(total, units, unit), end = unit_start(total, units, unit + 1);
    a.table[start + begin] = {(r << a.log_g) + g, end - begin, unit | (units << 16), first_slot(start)};
  }
}

// The units that begin at eight positions of the list: each thread a piece of the
// columns, all positions one after the other.
template <int FMT, int E>
__global__ __launch_bounds__(256) void embed_sum_kernel(EmbedGradArgs a) {
  __shared__ Unit s_unit[kRun];
  __shared__ bool s_last;
  static_assert(kRun <= kUnit / 2 && kFew <= 2 * kUnit);
  const int t = threadIdx.x, lane = t & 63, b = blockIdx.y * blockDim.x + t;
  const bool some = E * b < a.C;
  const int col = (some ? piece_at<FMT, E>(b, a.C) : 0) * kLogitBytes<FMT>;
  const int p0 = blockIdx.x * kRun, there = min((int64_t)kRun, a.N - p0);
  Unit own = {-1, 0, 0, 0};
  if (lane < there) own = a.table[p0 + lane];
  const uint32_t begin = (uint32_t)__ballot(own.row >= 0);
  if (begin == 0u) return;  // (the same for all waves)
  if (t < kRun) s_unit[t] = own;
  const int from = __builtin_ctz(begin), last_at = 31 - __builtin_clz(begin);
  const int n = last_at - from + __builtin_amdgcn_readlane(own.count, last_at);  // <= kRun - 1 + kUnit positions,
  const int pos = a.order[p0 + from + min(lane, n - 1)];                         // or one long unit's: 64 at a time
  __syncthreads();
  const char *dy = static_cast<const char *>(a.dy);
  float acc[E] = {};

  auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };  // (every lane has the same)
  auto put = [&](int row) {
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= a.scale;
    if (some) store_piece<FMT, E>(static_cast<char *>(a.out) + row * (int64_t)a.C * kLogitBytes<FMT> + col, acc);
  };
  Piece<FMT, E> x[kRun];
  auto load = [&](int lanes, int j, int to) {
    asm volatile("" : "+v"(lanes));  // (has arrived here: else each readlane below waits for the rows before it)
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      x[i] = {};
      if (j + i < to) x[i].load(dy + (int64_t)__builtin_amdgcn_readlane(lanes, j + i) * a.ldg * kLogitBytes<FMT> + col);
    }
  };
  auto add = [&](const Piece<FMT, E> &p) {
    float f[E];
    p.get(f);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += f[e];
  };

  // the first eight, where units begin; then what is left of the last one. (One of several
  // of its row has 16 positions or more: it can only be the last.)
  load(pos, 0, n);
  int at = from;
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    if (i > 0 && from + i < kRun && ((begin >> (from + i)) & 1u)) {
      put(uniform(s_unit[at].row));
      at = from + i;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
    }
    add(x[i]);
  }
  for (int j = kRun; j < n; j += kRun) {
    int lanes = pos;
    if (j >= kWave) lanes = a.order[p0 + from + min(j / kWave * kWave + lane, n - 1)];
    load(lanes, j % kWave, min(n - j / kWave * kWave, kWave));
#pragma unroll
    for (int i = 0; i < kRun; ++i) add(x[i]);
  }
  const Unit u = {uniform(s_unit[at].row), 0, uniform(s_unit[at].at), uniform(s_unit[at].slot)};
  const int units = u.at >> 16;
  if (units > 1) {
    // The sums as the units' threads have them: value e of all threads side by side.
    const int64_t unit_size = (int64_t)a.blocks * blockDim.x * E;
    float *part = a.part + u.slot * unit_size + (int64_t)blockIdx.y * blockDim.x * E + t;
    // stored past the caches of this XCD, acknowledged before the count goes up
#pragma unroll
    for (int e = 0; e < E; ++e)
      __hip_atomic_store(part + (u.at & 0xffff) * unit_size + e * blockDim.x, acc[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t == 0)
      s_last = __hip_atomic_fetch_add(a.arrived + (int64_t)u.slot * a.blocks + blockIdx.y, 1, __ATOMIC_RELAXED,
                                      __HIP_MEMORY_SCOPE_AGENT) == units - 1;
    __syncthreads();
    if (!s_last) return;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int i = 0; i < units; i += kJoin) {
      float p[kJoin][E];
#pragma unroll
      for (int k = 0; k < kJoin; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e)
          p[k][e] = __hip_atomic_load(part + min(i + k, units - 1) * unit_size + e * blockDim.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
      for (int k = 0; k < kJoin; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += i + k < units ? p[k][e] : 0.f;
    }
  }
  put(u.row);
}

int log_groups(int V) {
  int l = 8;
  while ((int64_t)kSortRows << l < V) ++l;
  return l;
}

// f(FMT, E) for a type and width
template <class F>
void with_pieces(int dtype, int C, F f) {
  using std::integral_constant;
  auto width = [&](auto fmt) {
    constexpr int FMT = decltype(fmt)::value;
    if (C >= kWide<FMT>) f(fmt, integral_constant<int, kWide<FMT>>());
    else f(fmt, integral_constant<int, 1>());
  };
  if (dtype == 0) width(integral_constant<int, 0>());
  else if (dtype == 1) width(integral_constant<int, 1>());
  else width(integral_constant<int, 2>());
}

// The sums' workgroups: a piece a thread, up to 256 threads.
struct SumShape {
  int threads, blocks, columns;
};
SumShape sum_shape(int dtype, int C) {
  SumShape s;
  with_pieces(dtype, C, [&](auto, auto e) {
    constexpr int E = decltype(e)::value;
    const int n = (pieces<E>(C) + kWave - 1) / kWave * kWave;
    s.threads = n < 256 ? n : 256;
    s.blocks = (n + s.threads - 1) / s.threads;
    s.columns = s.blocks * s.threads * E;
  });
  return s;
}

struct GradSpace {
  int64_t table, arrived, order, part, bytes;
};
GradSpace grad_space(int64_t N, int C, int dtype) {
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  GradSpace s = {};
  s.arrived = s.table + up(N * (int64_t)sizeof(Unit));
  s.order = s.arrived + up(slots(N) * sum_shape(dtype, C).blocks * 4);
  s.part = s.order + up(N * 4);
  s.bytes = s.part + slots(N) * sum_shape(dtype, C).columns * 4;
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
  with_pieces(dtype, C, [&](auto f, auto e) {
    embed_kernel<decltype(f)::value, decltype(e)::value><<<(int)((N + 3) / 4), 256, 0, st>>>(g);
  });
  RWKV7_CHECK_LAUNCH();
  return RWKV7_OK;
}

extern "C" int64_t rwkv7_embed_backward_workspace_bytes(int32_t dtype, int64_t N, int32_t V, int32_t C) {
  using namespace rwkv7;
  return sizes_ok(N, V, C) && dtype >= 0 && dtype <= 2 ? grad_space(N, C, dtype).bytes : 0;
}

extern "C" int rwkv7_embed_backward(const void *grad, int32_t dtype, int64_t ldg, const int64_t *tokens, float scale,
                                    void *grad_weight, int64_t N, int32_t V, int32_t C, void *workspace,
                                    int64_t workspace_bytes, void *stream) {
  using namespace rwkv7;
  if (!grad || !tokens || !grad_weight || !workspace || dtype < 0 || dtype > 2) return RWKV7_EINVAL;
  if (!sizes_ok(N, V, C) || ldg < C) return RWKV7_ESHAPE;
  const GradSpace s = grad_space(N, C, dtype);
  if (workspace_bytes < s.bytes) return RWKV7_EWORKSPACE;
  char *ws = static_cast<char *>(workspace);
  const SumShape shape = sum_shape(dtype, C);
  const EmbedGradArgs a = {grad, ldg, tokens, grad_weight, N, V, C, log_groups(V), scale, reinterpret_cast<int *>(ws + s.order),
                           reinterpret_cast<Unit *>(ws + s.table), reinterpret_cast<int *>(ws + s.arrived),
                           reinterpret_cast<float *>(ws + s.part), shape.blocks};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t fill = ((int64_t)V * C * logit_bytes(dtype) + kFillBytes - 1) / kFillBytes;
  const int groups = (1 << a.log_g) + (int)(fill < kFillGroups ? fill : kFillGroups);
  const bool held = N <= kHeld * kSortThreads;
  if (dtype == 1) {
    if (held) embed_sort_kernel<4, true><<<groups, kSortThreads, 0, st>>>(a);
    else embed_sort_kernel<4, false><<<groups, kSortThreads, 0, st>>>(a);
  } else {
    if (held) embed_sort_kernel<2, true><<<groups, kSortThreads, 0, st>>>(a);
    else embed_sort_kernel<2, false><<<groups, kSortThreads, 0, st>>>(a);
  }
  RWKV7_CHECK_LAUNCH();
  const dim3 grid((unsigned)((N + kRun - 1) / kRun), shape.blocks);
  with_pieces(dtype, C, [&](auto f, auto e) {
    embed_sum_kernel<decltype(f)::value, decltype(e)::value><<<grid, shape.threads, 0, st>>>(a);
  });
  RWKV7_CHECK_LAUNCH();
  return RWKV7_OK;
}
