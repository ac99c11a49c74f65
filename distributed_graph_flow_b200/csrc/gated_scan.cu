// Gated linear recurrence over ragged windows (sm_100a).
//
// For every segment s (rows off[s] .. off[s+1] of x and gate) and channel:
//   a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,
//   h before the first row = initial[s] (0 without it), final[s] = last h.
// Backward, with d_t the gradient of h_t and f[s] that of final[s]: let
// e_t = a_t delta_t be what flows to h_{t-1}; then e is itself such a
// recurrence run upwards,
//   delta_t = d_t + e_{t+1},  e_t = a_t (d_t + e_{t+1}),  e after the last
//   row = f[s];  dx_t = (1 - a_t) delta_t,
//   dgate_t = delta_t (h_{t-1} - x_t) a_t (1 - a_t),  dinitial[s] = e_first.
//
// All rows form one flat scan that restarts at the first row of a segment,
// cut into chunks of equal height whatever the windows' lengths, so the work
// balances. A thread owns two adjacent channels of one chunk and walks its rows one by
// one, the next rows' loads in flight; neighbouring threads are neighbouring channels,
// so loads and stores are whole rows, and nothing is shared between threads.
//
//   edge kernel    where each chunk's edge row stands among the segments;
//                  outputs of the segments without rows.
//   chunk kernel   what a chunk does to a state that passes through its last
//                  row: (A, H), state -> A state + H. Only the segment that crosses
//                  that edge matters, so only its rows in the chunk are read:
//                  a few rows where windows are short, all of them inside of
//                  a long one. A < 0 marks a segment that began in the chunk:
//                  the outgoing state is H alone (selected, not multiplied: a
//                  NaN of one window never reaches the next).
//   level kernel   (A, H) of groups of 32 chunks and of supergroups of 32
//                  groups; a chunk's place takes what comes before it in its
//                  group, a group's what comes before it in its supergroup.
//   apply kernel   composes the state that enters its chunk from those two
//                  and the supergroups since the segment began, then walks
//                  the rows and writes. No thread waits for another.
//
// Bound by HBM: one read of each input and one write of each output where
// windows are short, and up to a second read of gate and x (gate and grad,
// going backward) inside of windows longer than a chunk. The composition's
// shape depends on the sizes alone, so results do not change from run to run.
//
// Going backward, h is not read but computed again, from states that the
// forward pass saves before every kBlock-th row (4 bytes per kBlock rows and
// channel), in registers.
//
// States, products and gradients of states are fp32; h, dx and dgate are
// rounded once when written. Rows outside [off[0], off[nseg]) are written as
// zeros and their inputs are never used.
//
// Measured (L2 flushed): 20,000 windows of Zipf lengths in 600,011 rows x 64
// bf16 channels, forward 100 us, of which the apply kernel 55 (4.2 TB/s); 30,000
// windows in 1,200,007 rows x 128 bf16, forward + backward 650 us (apply 200 and
// 350: 1.0 GB at 5 TB/s, 1.6 GB at 4.6); 3 series of 393,209 rows x 96 fp32, forward +
// backward 361 us (apply 80 and 140 at 6.1 and 5.7 TB/s, chunk kernels 64 and 58: inside of long
// windows the inputs are read twice). What is left above HBM: the two special
// functions and some sixty instructions per channel pair and row.
#include <algorithm>
#include <string>

#include "layer_math.cuh"

namespace dgfx {
namespace {

constexpr int kThreads = 256;
constexpr int kApplyThreads = 128;
constexpr int kAhead = 1;  // blocks of rows on their way in the apply kernels
constexpr int kCh = 4;     // channels per thread of the single step
// Rows loaded at a time (32 bytes of each input); rows between saved states.
template <class T>
constexpr int kBlock = sizeof(T) == 2 ? 8 : 4;
constexpr int kLevel = 32;
constexpr int kSms = 148;

// Two adjacent values of T as fp32.
template <class T>
struct Pair;
template <>
struct Pair<float> {
  using raw = float2;
  __device__ static __forceinline__ float2 unpack(raw r) { return r; }
  __device__ static __forceinline__ raw pack(float2 f) { return f; }
  __device__ static __forceinline__ raw zero() { return make_float2(0.0f, 0.0f); }
};
template <>
struct Pair<__nv_bfloat16> {
  using raw = uint32_t;
  __device__ static __forceinline__ float2 unpack(raw r) {
    return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xFFFF0000u));
  }
  __device__ static __forceinline__ raw pack(float2 f) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static __forceinline__ raw zero() { return 0u; }
};

// a = sigmoid(g) and 1 - a = e^-g a, neither from a subtraction. The exponent
// is held above -80, where a is 2e-35, so that e^-g stays finite (a maximum
// that keeps NaN).
__device__ __forceinline__ void gate_pair(float g, float* a, float* keep) {
  float low;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(low) : "f"(g), "f"(-80.0f));
  const float e = exp_f(-low);
  *a = rcp_f(1.0f + e);
  *keep = e * *a;
}

// One row's coefficients and inputs for two channels.
template <class T>
struct Row {
  float2 a, keep, x;
  __device__ __forceinline__ Row(typename Pair<T>::raw gate, typename Pair<T>::raw in) {
    const float2 g = Pair<T>::unpack(gate);
    x = Pair<T>::unpack(in);
    gate_pair(g.x, &a.x, &keep.x);
    gate_pair(g.y, &a.y, &keep.y);
  }
  __device__ __forceinline__ void step(float2& h) const {
    h.x = fmaf(a.x, h.x, keep.x * x.x);
    h.y = fmaf(a.y, h.y, keep.y * x.y);
  }
};

struct Params {
  const void* x;
  const void* gate;
  const int64_t* off;
  const float* initial;
  const void* grad;
  const float* grad_final;
  void* h;
  float* final;
  void* dx;
  void* dgate;
  float* dinitial;
  float* save;         // forward: states before every kBlock-th row [ceil(rows / kBlock), channels], or null
  const float* saved;  // backward: the same
  float4* chunk_ah;    // (A, H, A, H) of two channels: [chunks, pairs]
  float4* group_ah;    // [groups, pairs]
  float4* super_ah;    // [supergroups, pairs]
  int32_t* first_seg;  // at a segment's first row: its number (other rows are not written) [rows]
  int32_t* last_seg;   // backward: the same at its last row
  int32_t* edge_seg;   // per chunk: where its first (backward: last) row stands among the segments [chunks]
  int64_t rows, nseg, chunks, groups, supers;
  int32_t channels, pairs, chunk_rows, chunk_shift;  // chunk_rows = 1 << chunk_shift
};

// (A, H) of two channels.
struct Effect {
  float4 v;
  __device__ Effect() : v(make_float4(1.0f, 0.0f, 1.0f, 0.0f)) {}
  __device__ void then(const float4& n) {
    v.y = n.x < 0.0f ? n.y : fmaf(n.x, v.y, n.y);
    v.w = n.z < 0.0f ? n.w : fmaf(n.z, v.w, n.w);
    v.x = (n.x < 0.0f || v.x < 0.0f) ? -1.0f : v.x * n.x;
    v.z = (n.z < 0.0f || v.z < 0.0f) ? -1.0f : v.z * n.z;
  }
};

__device__ __forceinline__ float2 load2(const float* base, int64_t row, int channels, int ch) {
  return __ldg(reinterpret_cast<const float2*>(base + row * channels + ch));
}
__device__ __forceinline__ void store2(float* base, int64_t row, int channels, int ch, float2 v) {
  *reinterpret_cast<float2*>(base + row * channels + ch) = v;
}

// Chunk and pair of this thread (32-bit division where the grid allows).
struct Spot {
  int64_t j;
  int pair, ch;
  __device__ explicit Spot(const Params& p) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (t <= 0x7fffffff) {
      const uint32_t q = static_cast<uint32_t>(t) / static_cast<uint32_t>(p.pairs);
      j = q;
      pair = static_cast<int>(static_cast<uint32_t>(t) - q * static_cast<uint32_t>(p.pairs));
    } else {
      j = t / p.pairs;
      pair = static_cast<int>(t - j * p.pairs);
    }
    ch = 2 * pair;
  }
};

// This thread's column of an input or output, from row r0.
template <class T>
__device__ __forceinline__ const typename Pair<T>::raw* column(const void* base, const Params& p, int64_t r0, int pair) {
  return static_cast<const typename Pair<T>::raw*>(base) + r0 * p.pairs + pair;
}
template <class T>
__device__ __forceinline__ typename Pair<T>::raw* column(void* base, const Params& p, int64_t r0, int pair) {
  return static_cast<typename Pair<T>::raw*>(base) + r0 * p.pairs + pair;
}

// ---------------------------------------------------------------------------
// Edge kernel: a warp per segment
// ---------------------------------------------------------------------------
// Forward, edge_seg[j] = the segment of chunk j's first row: -1 before the
// first segment, nseg behind the last. Backward, the last segment with rows
// that begins at or before chunk j's last row, -1 if there is none. Every
// segment with rows leaves its number at its first row (backward: and at its
// last), so that a walk steps from one to the next by one load, however many
// segments without rows lie between them (searching the offsets there took
// 106 us at 2269 windows of 124 rows). Segments without rows get their state or
// gradient of it: out[s] = in[s] (0 without `in`).
__global__ void __launch_bounds__(kThreads) scan_edge_kernel(Params p, int up, const float* __restrict__ in,
                                                             float* __restrict__ out) {
  let_next_start();
  const int64_t threads = static_cast<int64_t>(gridDim.x) * kThreads;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int lane = threadIdx.x & 31;
  const int64_t lo = clamp64(__ldg(p.off), 0, p.rows), hi = clamp64(__ldg(p.off + p.nseg), lo, p.rows);
  for (int64_t j = t; j < p.chunks; j += threads) {
    const int64_t first = j << p.chunk_shift, next = first + p.chunk_rows;
    if (up) {
      if ((next < p.rows ? next : p.rows) <= lo || lo == hi) p.edge_seg[j] = -1;
    } else if (first < lo || first >= hi) {
      p.edge_seg[j] = first < lo ? -1 : static_cast<int32_t>(p.nseg);
    }
  }
  for (int64_t s = t >> 5; s < p.nseg; s += threads >> 5) {
    const int64_t b = clamp64(__ldg(p.off + s), lo, hi), e = clamp64(__ldg(p.off + s + 1), b, hi);
    if (b == e) {
      if (out != nullptr) {
        for (int c = 2 * lane; c < p.channels; c += 64) {
          store2(out, s, p.channels, c, in != nullptr ? load2(in, s, p.channels, c) : make_float2(0.0f, 0.0f));
        }
      }
      continue;
    }
    if (lane == 0) {
      p.first_seg[b] = static_cast<int32_t>(s);
      if (up) p.last_seg[e - 1] = static_cast<int32_t>(s);
    }
    if (up) {
      // Chunks whose last row lies in [b, e); of the last segment with rows,
      // also the chunks behind it.
      for (int64_t j = (b >> p.chunk_shift) + lane; j < p.chunks; j += 32) {
        const int64_t next = (j + 1) << p.chunk_shift;
        if (e != hi && (next < p.rows ? next : p.rows) > e) break;
        p.edge_seg[j] = static_cast<int32_t>(s);
      }
    } else {
      for (int64_t j = ((b + p.chunk_rows - 1) >> p.chunk_shift) + lane; (j << p.chunk_shift) < e; j += 32) {
        p.edge_seg[j] = static_cast<int32_t>(s);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Chunk kernels
// ---------------------------------------------------------------------------
// Calls f for n rows from `gate` and `in` on (null: zeros), `pitch` apart, in
// order; the next block's loads are on their way while this one's run.
template <class T, class F>
__device__ __forceinline__ void walk(const typename Pair<T>::raw* gate, const typename Pair<T>::raw* in, int pitch, int n,
                                     F f) {
  constexpr int B = kBlock<T>;
  using raw = typename Pair<T>::raw;
  raw g[B], x[B];
  auto fetch = [&](int left, raw(&gv)[B], raw(&xv)[B]) {  // the next block, `left` rows from the end
#pragma unroll
    for (int i = 0; i < B; ++i) {
      gv[i] = i < left ? __ldg(gate + i * pitch) : Pair<T>::zero();
      xv[i] = i < left && in != nullptr ? __ldg(in + i * pitch) : Pair<T>::zero();
    }
    gate += B * pitch;
    if (in != nullptr) in += B * pitch;
  };
  fetch(n, g, x);
  for (int left = n; left > 0; left -= B) {
    raw gn[B], xn[B];
    fetch(left - B, gn, xn);
    if (left >= B) {
#pragma unroll
      for (int i = 0; i < B; ++i) f(Row<T>(g[i], x[i]));
    } else {
#pragma unroll
      for (int i = 0; i < B; ++i) {
        if (i < left) f(Row<T>(g[i], x[i]));
      }
    }
#pragma unroll
    for (int i = 0; i < B; ++i) {
      g[i] = gn[i];
      x[i] = xn[i];
    }
  }
}

// Forward: thread (j, pair) writes the effect of chunk j on the segment that
// crosses its lower edge, the first row of chunk j + 1.
template <class T>
__global__ void __launch_bounds__(kThreads, 4) scan_chunk_kernel(Params p) {
  let_next_start();
  after_previous();
  const Spot at(p);
  if (at.j + 1 >= p.chunks) return;
  const int64_t first = at.j << p.chunk_shift, edge = first + p.chunk_rows;
  // Clamped here and below: offsets that do not ascend leave anything.
  const int64_t seg = clamp64(p.edge_seg[at.j + 1], -1, p.nseg);
  Effect f;
  f.v = make_float4(-1.0f, 0.0f, -1.0f, 0.0f);
  if (seg >= 0 && seg < p.nseg) {
    const int64_t begin = __ldg(p.off + seg);
    const int64_t from = clamp64(begin, first, edge);
    const int n = static_cast<int>(edge - from);
    if (n > 0) {
      float2 a = make_float2(1.0f, 1.0f), h = make_float2(0.0f, 0.0f);
      if (begin >= first && p.initial != nullptr) h = load2(p.initial, seg, p.channels, at.ch);
      walk<T>(column<T>(p.gate, p, from, at.pair), column<T>(p.x, p, from, at.pair), p.pairs, n, [&](const Row<T>& row) {
        row.step(h);
        a.x *= row.a.x;
        a.y *= row.a.y;
      });
      const bool began = begin >= first;
      f.v = make_float4(began ? -1.0f : a.x, h.x, began ? -1.0f : a.y, h.y);
    }
  }
  p.chunk_ah[at.j * p.pairs + at.pair] = f.v;
}

// Backward: the effect of chunk j, upwards, on the segment that crosses its
// upper edge.
template <class T>
__global__ void __launch_bounds__(kThreads, 4) scan_chunk_up_kernel(Params p) {
  let_next_start();
  after_previous();
  const Spot at(p);
  if (at.j >= p.chunks || at.j == 0) return;
  const int64_t edge = at.j << p.chunk_shift;
  const int64_t stop = edge + p.chunk_rows < p.rows ? edge + p.chunk_rows : p.rows;
  // The segment of the last row above the edge, if it goes on below it.
  const int64_t seg = clamp64(p.edge_seg[at.j - 1], -1, p.nseg - 1);
  Effect f;
  f.v = make_float4(-1.0f, 0.0f, -1.0f, 0.0f);
  if (seg >= 0 && __ldg(p.off + seg + 1) > edge) {
    const int64_t end = __ldg(p.off + seg + 1);
    const int n = static_cast<int>(clamp64(end, edge, stop) - edge);
    float2 a = make_float2(1.0f, 1.0f), e = make_float2(0.0f, 0.0f);
    if (end <= stop && p.grad_final != nullptr) e = load2(p.grad_final, seg, p.channels, at.ch);
    const auto* dp = p.grad != nullptr ? column<T>(p.grad, p, edge + n - 1, at.pair) : nullptr;
    walk<T>(column<T>(p.gate, p, edge + n - 1, at.pair), dp, -p.pairs, n, [&](const Row<T>& row) {
      e.x = row.a.x * (row.x.x + e.x);
      e.y = row.a.y * (row.x.y + e.y);
      a.x *= row.a.x;
      a.y *= row.a.y;
    });
    const bool ended = end <= stop;
    f.v = make_float4(ended ? -1.0f : a.x, e.x, ended ? -1.0f : a.y, e.y);
  }
  p.chunk_ah[at.j * p.pairs + at.pair] = f.v;
}

// Every item of a level becomes the effect of the items of its group (kLevel
// of them) before it, in the order of the pass (`up`: from the last to the
// first); out[g] is the effect of group g. Sixteen loads in flight.
__global__ void __launch_bounds__(kThreads) scan_level_kernel(float4* items, int64_t count, int pairs, int up, float4* out,
                                                              int64_t outs) {
  let_next_start();
  after_previous();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t g = t / pairs;
  const int pair = static_cast<int>(t - g * pairs);
  if (g >= outs) return;
  const int64_t first = g * kLevel, last = first + kLevel < count ? first + kLevel : count;
  float4* item = items + (up ? last - 1 : first) * pairs + pair;
  const int64_t step = up ? -pairs : pairs;
  const int n = static_cast<int>(last - first);
  Effect f;
  for (int i = 0; i < n; i += kLevel / 2) {
    float4 v[kLevel / 2];
#pragma unroll
    for (int k = 0; k < kLevel / 2; ++k) {
      if (i + k < n) v[k] = item[k * step];
    }
#pragma unroll
    for (int k = 0; k < kLevel / 2; ++k) {
      if (i + k < n) {
        item[k * step] = f.v;
        f.then(v[k]);
      }
    }
    item += kLevel / 2 * step;
  }
  out[g * pairs + pair] = f.v;
}

// The state that enters chunk j when the segment at its edge began in chunk
// o < j (going up: ends in chunk o > j): the supergroups from o's on, then
// the groups before j's in its own, then the chunks before j in its own.
// What they hold of other segments ends where that one begins. Up to kLevel
// chunks are composed as they are: the level kernels' launches took 2 us more
// there (96 rows: 22.6 against 26.6 us).
__device__ __forceinline__ float2 entering(const Params& p, int64_t j, int64_t o, int pair) {
  Effect f;
  if (p.groups == 1) {  // no level kernel ran
    constexpr int N = 8;
    const int64_t step = o < j ? p.pairs : -p.pairs;
    const float4* item = p.chunk_ah + o * p.pairs + pair;
    for (int left = static_cast<int>(o < j ? j - o : o - j); left > 0; left -= N) {
      float4 v[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if (k < left) v[k] = item[k * step];
      }
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if (k < left) f.then(v[k]);
      }
      item += N * step;
    }
    return make_float2(f.v.y, f.v.w);
  }
  const int64_t g = j / kLevel, s = g / kLevel;
  const float4 chunk = p.chunk_ah[j * p.pairs + pair], group = p.group_ah[g * p.pairs + pair];
  for (int64_t so = o / kLevel / kLevel; so != s; so += so < s ? 1 : -1) f.then(p.super_ah[so * p.pairs + pair]);
  f.then(group);
  f.then(chunk);
  return make_float2(f.v.y, f.v.w);
}

// ---------------------------------------------------------------------------
// Apply kernels
// ---------------------------------------------------------------------------
// Both walk a chunk in blocks of kBlock rows, the loads of the next kAhead
// blocks in flight on their way to shared memory, where each thread has slots
// of its own: they cost no registers (held in registers instead, 80 bytes
// spilled and a long series took 91 rather than 80 us). One block ahead is
// enough: two and three measured 57 and 62 us at 600,011 rows of 64 channels,
// one 55. A block that lies inside of one segment, with neither edge of it,
// takes the plain path; any other is walked with its checks per row.
// A thread waits for its own copies only.
template <class T, int INPUTS>
struct Slots {
  static constexpr int B = kBlock<T>;
  using raw = typename Pair<T>::raw;
  raw v[kAhead + 1][INPUTS][B][kApplyThreads];

  // Starts on rows of one input, `pitch` apart, into a stage; `left` of them
  // are there, the others read as zeros.
  __device__ __forceinline__ void start(int stage, int input, const raw* from, int pitch, int left) {
    raw* to = &v[stage][input][0][threadIdx.x];
    if (left >= B) {
#pragma unroll
      for (int i = 0; i < B; ++i) copy(to + i * kApplyThreads, from + i * pitch);
    } else {
#pragma unroll
      for (int i = 0; i < B; ++i) {
        if (i < left) copy(to + i * kApplyThreads, from + i * pitch);
        else to[i * kApplyThreads] = Pair<T>::zero();
      }
    }
  }
  __device__ static __forceinline__ void copy(raw* to, const raw* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(to))),
                 "l"(from), "n"(sizeof(raw))
                 : "memory");
  }
  // Closes the block that was started last; waits for the one kAhead blocks
  // before it.
  __device__ static __forceinline__ void close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  __device__ static __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory"); }
  __device__ __forceinline__ raw get(int stage, int input, int i) const { return v[stage][input][i][threadIdx.x]; }
};

template <class T>
__global__ void __launch_bounds__(kApplyThreads, 8) scan_apply_kernel(Params p) {
  after_previous();
  constexpr int B = kBlock<T>;
  using P = Pair<T>;
  using raw = typename P::raw;
  __shared__ Slots<T, 2> slots;
  const Spot at(p);
  if (at.j < p.chunks) {
    const int64_t r0 = at.j << p.chunk_shift;
    const int n = static_cast<int>(p.rows - r0 < p.chunk_rows ? p.rows - r0 : p.chunk_rows);
    const raw* gp = column<T>(p.gate, p, r0, at.pair);
    const raw* xp = column<T>(p.x, p, r0, at.pair);
    raw* hp = p.h != nullptr ? column<T>(p.h, p, r0, at.pair) : nullptr;
    auto start = [&](int stage, int left) {  // the next block, `left` rows from the end
      if (left > 0) {
        slots.start(stage, 0, gp, p.pairs, left);
        slots.start(stage, 1, xp, p.pairs, left);
        gp += B * p.pairs;
        xp += B * p.pairs;
      }
      slots.close();
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k) start(k, n - k * B);
    int stage = 0;
    // The current segment, the row (from r0) where it ends, and whether there
    // is one: rows before the first and behind the last have none.
    int64_t seg = clamp64(p.edge_seg[at.j], -1, p.nseg);
    const int64_t hi = clamp64(__ldg(p.off + p.nseg), 0, p.rows);
    auto until = [&](int64_t row) { return static_cast<int>(clamp64(row - r0, 0, p.chunk_rows + 1)); };
    bool inside = seg >= 0 && seg < p.nseg;
    int limit;
    float2 st = make_float2(0.0f, 0.0f);
    if (inside) {
      const int64_t begin = clamp64(__ldg(p.off + seg), 0, r0);
      limit = until(__ldg(p.off + seg + 1));
      if (begin < r0) st = entering(p, at.j, begin >> p.chunk_shift, at.pair);
      else if (p.initial != nullptr) st = load2(p.initial, seg, p.channels, at.ch);
    } else {
      limit = seg < 0 ? until(__ldg(p.off)) : p.chunk_rows + 1;
    }
    if (limit == 0) limit = p.chunk_rows + 1;  // only where offsets do not ascend
    float* save = p.save != nullptr ? p.save + r0 / B * p.channels + at.ch : nullptr;
    for (int b0 = 0; b0 < n; b0 += B) {
      start(stage == 0 ? kAhead : stage - 1, n - b0 - kAhead * B);
      slots.wait();
      if (save != nullptr) {
        *reinterpret_cast<float2*>(save) = st;
        save += p.channels;
      }
      if (inside && b0 + B < limit && b0 + B <= n) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
          const Row<T> row(slots.get(stage, 0, i), slots.get(stage, 1, i));
          row.step(st);
          if (hp != nullptr) hp[i * p.pairs] = P::pack(st);
        }
      } else {
#pragma unroll
        for (int i = 0; i < B; ++i) {
          const int r = b0 + i;
          if (r < n) {
            const Row<T> row(slots.get(stage, 0, i), slots.get(stage, 1, i));
            row.step(st);
            if (!inside) st = make_float2(0.0f, 0.0f);
            if (hp != nullptr) hp[i * p.pairs] = P::pack(st);
            if (r + 1 == limit) {  // this row is the segment's last: on to the next one with rows
              if (inside && p.final != nullptr) store2(p.final, seg, p.channels, at.ch, st);
              seg = r0 + r + 1 < hi ? clamp64(p.first_seg[r0 + r + 1], 0, p.nseg - 1) : p.nseg;
              inside = seg < p.nseg;
              if (inside) {
                const int64_t end = __ldg(p.off + seg + 1);
                limit = until(end < hi ? end : hi);
              } else {
                limit = p.chunk_rows + 1;
              }
              st = inside && p.initial != nullptr ? load2(p.initial, seg, p.channels, at.ch) : make_float2(0.0f, 0.0f);
            }
          }
        }
      }
      if (hp != nullptr) hp += B * p.pairs;
      stage = stage == kAhead ? 0 : stage + 1;
    }
  }
}

template <class T>
__global__ void __launch_bounds__(kApplyThreads, 4) scan_apply_up_kernel(Params p) {
  after_previous();
  constexpr int B = kBlock<T>;
  using P = Pair<T>;
  using raw = typename P::raw;
  __shared__ Slots<T, 3> slots;
  const Spot at(p);
  if (at.j < p.chunks) {
    const int64_t r0 = at.j << p.chunk_shift;
    const int n = static_cast<int>(p.rows - r0 < p.chunk_rows ? p.rows - r0 : p.chunk_rows);
    const int64_t lo64 = clamp64(__ldg(p.off), 0, p.rows), hi64 = clamp64(__ldg(p.off + p.nseg), lo64, p.rows);
    auto rel = [&](int64_t row) { return static_cast<int>(clamp64(row - r0, -1, p.chunk_rows + 1)); };
    const int lo = rel(lo64), hi = rel(hi64);
    int b0 = (n - 1) / B * B;
    const raw* gp = column<T>(p.gate, p, r0 + b0, at.pair);
    const raw* xp = column<T>(p.x, p, r0 + b0, at.pair);
    const raw* dp = p.grad != nullptr ? column<T>(p.grad, p, r0 + b0, at.pair) : nullptr;
    raw* dxp = column<T>(p.dx, p, r0 + b0, at.pair);
    raw* dgp = column<T>(p.dgate, p, r0 + b0, at.pair);
    auto start = [&](int stage, int left) {  // the next block up, `left` rows from the end (none: no such block)
      if (left > 0) {
        slots.start(stage, 0, gp, p.pairs, left);
        slots.start(stage, 1, xp, p.pairs, left);
        if (dp != nullptr) slots.start(stage, 2, dp, p.pairs, left);
        gp -= B * p.pairs;
        xp -= B * p.pairs;
        if (dp != nullptr) dp -= B * p.pairs;
      }
      slots.close();
    };
    start(0, n - b0);
#pragma unroll
    for (int k = 1; k < kAhead; ++k) start(k, b0 >= k * B ? B : 0);
    int stage = 0;
    const float* saved = p.saved + (r0 + b0) / B * p.channels + at.ch;
    float2 before = __ldg(reinterpret_cast<const float2*>(saved));
    // The segment of the current row (with rows; -1 when none is left), its
    // first row and the row behind its last, from r0.
    int64_t seg = clamp64(p.edge_seg[at.j], -1, p.nseg - 1);
    int begin = seg >= 0 ? rel(__ldg(p.off + seg)) : -1;
    int end = seg >= 0 ? rel(__ldg(p.off + seg + 1)) : -1;
    // The segment with rows before the one that begins at row b. (Offsets that
    // do not ascend may name one that is not above it: the walk ends there.)
    auto step_back = [&](int b, int64_t* to, int* to_begin) {
      *to = r0 + b > lo64 && r0 + b <= p.rows ? clamp64(p.last_seg[r0 + b - 1], 0, p.nseg - 1) : -1;
      *to_begin = *to >= 0 ? rel(__ldg(p.off + *to)) : -1;
      if (*to_begin >= b) *to = *to_begin = -1;
    };
    float2 e = make_float2(0.0f, 0.0f);
    if (seg >= 0) {
      const int64_t end64 = clamp64(__ldg(p.off + seg + 1), 0, p.rows);
      if (end64 > r0 + n) e = entering(p, at.j, (end64 - 1) >> p.chunk_shift, at.pair);
    }
    for (; b0 >= 0; b0 -= B) {
      start(stage == 0 ? kAhead : stage - 1, b0 >= kAhead * B ? B : 0);
      slots.wait();
      float2 before_next = make_float2(0.0f, 0.0f);
      if (b0 > 0) {
        saved -= p.channels;
        before_next = __ldg(reinterpret_cast<const float2*>(saved));
      }
      float2 st = before;
      if (seg >= 0 && begin < b0 && end > b0 + B && b0 + B <= n) {
        float2 a[B], keep[B], q[B];  // q = (h_{t-1} - x_t) a_t (1 - a_t), forward
#pragma unroll
        for (int i = 0; i < B; ++i) {
          const Row<T> row(slots.get(stage, 0, i), slots.get(stage, 1, i));
          a[i] = row.a;
          keep[i] = row.keep;
          q[i] = make_float2((st.x - row.x.x) * (row.a.x * row.keep.x), (st.y - row.x.y) * (row.a.y * row.keep.y));
          row.step(st);
        }
#pragma unroll
        for (int i = B - 1; i >= 0; --i) {
          const float2 dv = P::unpack(dp != nullptr ? slots.get(stage, 2, i) : P::zero());
          const float2 delta = make_float2(dv.x + e.x, dv.y + e.y);
          e = make_float2(a[i].x * delta.x, a[i].y * delta.y);
          dxp[i * p.pairs] = P::pack(make_float2(keep[i].x * delta.x, keep[i].y * delta.y));
          dgp[i * p.pairs] = P::pack(make_float2(q[i].x * delta.x, q[i].y * delta.y));
        }
      } else {
        // Which rows of the block start a segment.
        uint32_t starts = 0;
        int64_t low = seg;
        int b = begin;
        while (low >= 0 && b >= b0) {
          if (b < b0 + B) starts |= 1u << (b - b0);
          step_back(b, &low, &b);
        }
        float2 a[B], keep[B], q[B];
#pragma unroll
        for (int i = 0; i < B; ++i) {
          if ((starts >> i) & 1u) {
            st = make_float2(0.0f, 0.0f);
            if (p.initial != nullptr) {
              st = load2(p.initial, clamp64(p.first_seg[r0 + b0 + i], 0, p.nseg - 1), p.channels, at.ch);
            }
          }
          const Row<T> row(slots.get(stage, 0, i), slots.get(stage, 1, i));
          a[i] = row.a;
          keep[i] = row.keep;
          q[i] = make_float2((st.x - row.x.x) * (row.a.x * row.keep.x), (st.y - row.x.y) * (row.a.y * row.keep.y));
          row.step(st);
        }
#pragma unroll
        for (int i = B - 1; i >= 0; --i) {
          const int r = b0 + i;
          if (r < n) {
            const bool inside = r >= lo && r < hi;
            if (r + 1 == end) {
              e = p.grad_final != nullptr ? load2(p.grad_final, seg, p.channels, at.ch) : make_float2(0.0f, 0.0f);
            }
            const float2 dv = P::unpack(dp != nullptr ? slots.get(stage, 2, i) : P::zero());
            const float2 delta = make_float2(dv.x + e.x, dv.y + e.y);
            const float2 dx = make_float2(keep[i].x * delta.x, keep[i].y * delta.y);
            const float2 dg = make_float2(q[i].x * delta.x, q[i].y * delta.y);
            e = inside ? make_float2(a[i].x * delta.x, a[i].y * delta.y) : make_float2(0.0f, 0.0f);
            dxp[i * p.pairs] = inside ? P::pack(dx) : P::zero();
            dgp[i * p.pairs] = inside ? P::pack(dg) : P::zero();
            if ((starts >> i) & 1u) {  // this row is the segment's first: on to the one before
              if (p.dinitial != nullptr) store2(p.dinitial, seg, p.channels, at.ch, e);
              step_back(r, &seg, &begin);
              end = seg >= 0 ? r : -1;
            }
          }
        }
      }
      dxp -= B * p.pairs;
      dgp -= B * p.pairs;
      stage = stage == kAhead ? 0 : stage + 1;
      before = before_next;
    }
  }
}

template <class T>
__global__ void scan_step_kernel(const typename Quad<T>::raw* __restrict__ x,
                                 const typename Quad<T>::raw* __restrict__ gate, const float4* state, int64_t n,
                                 typename Quad<T>::raw* __restrict__ h, float4* new_state) {
  using Q = Quad<T>;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const float4 s4 = state[i];
    float xv[kCh], gv[kCh], st[kCh] = {s4.x, s4.y, s4.z, s4.w};
    Q::unpack(__ldg(x + i), xv);
    Q::unpack(__ldg(gate + i), gv);
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      float av, keep;
      gate_pair(gv[c], &av, &keep);
      st[c] = fmaf(av, st[c], keep * xv[c]);
    }
    h[i] = Q::pack(st);
    new_state[i] = make_float4(st[0], st[1], st[2], st[3]);
  }
}

int check_shape(const char* who, int64_t rows, int64_t channels, int64_t nseg, int dtype) {
  if (rows < 0 || nseg < 0 || channels < kCh || channels % kCh != 0 || (dtype != DGFX_F32 && dtype != DGFX_BF16)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT,
                std::string(who) + ": need rows >= 0, segments >= 0, channels a positive multiple of 4, dtype fp32 or "
                                   "bf16");
  }
  if (channels > (int64_t(1) << 20) || nseg >= (int64_t(1) << 31) - 1 || rows > (int64_t(1) << 40) ||
      rows * channels > (int64_t(1) << 42)) {
    return fail(DGFX_ERR_UNSUPPORTED, std::string(who) + ": sizes out of range");
  }
  return DGFX_OK;
}

// Quads of x, gate, h and their gradients are loaded whole.
bool quad_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == DGFX_F32 ? 15u : 7u)) == 0;
}

// Chunk height (its logarithm): at least 16 rows, at most 256, and about 1024
// threads per SM in between. Lower chunks make the chunk kernel read more rows
// (1.2 million rows of 128 channels: 46 us at 128 rows, 37 at 256, 50 at 512, too
// few threads); at 512 threads per SM the apply kernel took 77 us instead of 58
// (600,011 rows of 64 channels), at 2048 the same.
int32_t chunk_shift_of(int64_t rows, int64_t channels) {
  const int64_t full = static_cast<int64_t>(kSms) * 1024;
  const int64_t want = rows * (channels / 2) / full;
  int32_t shift = 4;
  while (shift < 8 && (int64_t(1) << shift) < want) ++shift;
  return shift;
}

size_t carve(void* base, size_t cap, int64_t rows, int64_t channels, Params* p, bool* ok) {
  Arena arena(base, cap);
  p->rows = rows;
  p->channels = static_cast<int32_t>(channels);
  p->pairs = static_cast<int32_t>(channels / 2);
  p->chunk_shift = chunk_shift_of(rows, channels);
  p->chunk_rows = 1 << p->chunk_shift;
  p->chunks = ceil_div(rows, p->chunk_rows);
  p->groups = ceil_div(p->chunks, kLevel);
  p->supers = ceil_div(p->groups, kLevel);
  p->chunk_ah = arena.take<float4>(static_cast<size_t>(p->chunks) * p->pairs);
  p->group_ah = arena.take<float4>(static_cast<size_t>(p->groups) * p->pairs);
  p->super_ah = arena.take<float4>(static_cast<size_t>(p->supers) * p->pairs);
  p->edge_seg = arena.take<int32_t>(static_cast<size_t>(p->chunks));
  p->first_seg = arena.take<int32_t>(static_cast<size_t>(rows));
  p->last_seg = arena.take<int32_t>(static_cast<size_t>(rows));
  *ok = arena.ok();
  return arena.used;
}

unsigned grid_of(int64_t items, int threads = kThreads) {
  return static_cast<unsigned>(std::max<int64_t>(1, ceil_div(items, threads)));
}

template <class T>
int launch(const Params& p, bool up, cudaStream_t stream) {
  const unsigned grid = grid_of(p.chunks * p.pairs);
  const unsigned edges = grid_of(std::max(p.chunks, std::min<int64_t>(p.nseg * 32, kSms * 2048)));
  scan_edge_kernel<<<edges, kThreads, 0, stream>>>(p, up, up ? p.grad_final : p.initial, up ? p.dinitial : p.final);
  if (p.chunks > 1) {
    if (up) launch_after(scan_chunk_up_kernel<T>, grid, kThreads, 0, stream, p);
    else launch_after(scan_chunk_kernel<T>, grid, kThreads, 0, stream, p);
    // The forward pass has no edge behind the last chunk, the backward pass
    // none above the first: those effects are not written, and only reach
    // totals that nothing needs.
    if (p.groups > 1) {
      launch_after(scan_level_kernel, grid_of(p.groups * p.pairs), kThreads, 0, stream, p.chunk_ah, p.chunks, p.pairs, up,
                   p.group_ah, p.groups);
      launch_after(scan_level_kernel, grid_of(p.supers * p.pairs), kThreads, 0, stream, p.group_ah, p.groups, p.pairs, up,
                   p.super_ah, p.supers);
    }
  }
  if (p.chunks > 0) {
    const unsigned blocks = grid_of(p.chunks * p.pairs, kApplyThreads);
    if (up) launch_after(scan_apply_up_kernel<T>, blocks, kApplyThreads, 0, stream, p);
    else launch_after(scan_apply_kernel<T>, blocks, kApplyThreads, 0, stream, p);
  }
  DGFX_CUDA_TRY(cudaGetLastError());
  return DGFX_OK;
}

}  // namespace
}  // namespace dgfx

using namespace dgfx;

extern "C" int dgfx_gated_scan_workspace_size(int64_t rows, int64_t channels, int dtype, size_t* workspace_bytes,
                                              size_t* saved_bytes) {
  DGFX_TRY(check_shape("dgfx_gated_scan_workspace_size", rows, channels, 0, dtype));
  Params p{};
  bool ok;
  if (workspace_bytes != nullptr) *workspace_bytes = carve(nullptr, 0, rows, channels, &p, &ok);
  const int64_t block = dtype == DGFX_F32 ? kBlock<float> : kBlock<__nv_bfloat16>;
  if (saved_bytes != nullptr) *saved_bytes = static_cast<size_t>(ceil_div(rows, block)) * channels * sizeof(float);
  return DGFX_OK;
}

extern "C" int dgfx_gated_scan(const void* d_x, const void* d_gate, int dtype, int64_t rows, int64_t channels,
                               const int64_t* d_offsets, int64_t nseg, const float* d_initial, void* d_h,
                               float* d_final, float* d_saved, void* d_workspace, size_t workspace_bytes,
                               dgfx_stream stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  DGFX_TRY(check_shape("dgfx_gated_scan", rows, channels, nseg, dtype));
  if (d_offsets == nullptr || (rows > 0 && (d_x == nullptr || d_gate == nullptr))) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_scan: null operand");
  }
  if (!quad_aligned(d_x, dtype) || !quad_aligned(d_gate, dtype) || !quad_aligned(d_h, dtype) ||
      !quad_aligned(d_initial, DGFX_F32) || !quad_aligned(d_final, DGFX_F32) || !quad_aligned(d_saved, DGFX_F32)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_scan: operands must be aligned to 4 elements");
  }
  Params p{};
  bool ok = false;
  carve(d_workspace, workspace_bytes, rows, channels, &p, &ok);
  if (rows > 0 && (d_workspace == nullptr || !ok)) {
    return fail(DGFX_ERR_WORKSPACE, "dgfx_gated_scan: workspace too small");
  }
  if (rows > 0 && !ptr_aligned16(d_workspace)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_scan: the workspace must be 16-byte aligned");
  }
  p.x = d_x;
  p.gate = d_gate;
  p.off = d_offsets;
  p.initial = d_initial;
  p.h = d_h;
  p.final = d_final;
  p.save = d_saved;
  p.nseg = nseg;
  return dtype == DGFX_F32 ? launch<float>(p, false, stream) : launch<__nv_bfloat16>(p, false, stream);
}

extern "C" int dgfx_gated_scan_backward(const void* d_x, const void* d_gate, int dtype, int64_t rows, int64_t channels,
                                        const int64_t* d_offsets, int64_t nseg, const float* d_initial,
                                        const float* d_saved, const void* d_grad_h, const float* d_grad_final,
                                        void* d_dx, void* d_dgate, float* d_dinitial, void* d_workspace,
                                        size_t workspace_bytes, dgfx_stream stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  DGFX_TRY(check_shape("dgfx_gated_scan_backward", rows, channels, nseg, dtype));
  if (d_offsets == nullptr || (rows > 0 && (d_x == nullptr || d_gate == nullptr || d_saved == nullptr ||
                                            d_dx == nullptr || d_dgate == nullptr))) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_scan_backward: null operand");
  }
  if (!quad_aligned(d_x, dtype) || !quad_aligned(d_gate, dtype) || !quad_aligned(d_grad_h, dtype) ||
      !quad_aligned(d_dx, dtype) || !quad_aligned(d_dgate, dtype) || !quad_aligned(d_initial, DGFX_F32) ||
      !quad_aligned(d_saved, DGFX_F32) || !quad_aligned(d_grad_final, DGFX_F32) ||
      !quad_aligned(d_dinitial, DGFX_F32)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_scan_backward: operands must be aligned to 4 elements");
  }
  Params p{};
  bool ok = false;
  carve(d_workspace, workspace_bytes, rows, channels, &p, &ok);
  if (rows > 0 && (d_workspace == nullptr || !ok)) {
    return fail(DGFX_ERR_WORKSPACE, "dgfx_gated_scan_backward: workspace too small");
  }
  if (rows > 0 && !ptr_aligned16(d_workspace)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_scan_backward: the workspace must be 16-byte aligned");
  }
  p.x = d_x;
  p.gate = d_gate;
  p.off = d_offsets;
  p.initial = d_initial;
  p.grad = d_grad_h;
  p.grad_final = d_grad_final;
  p.dx = d_dx;
  p.dgate = d_dgate;
  p.dinitial = d_dinitial;
  p.saved = d_saved;
  p.nseg = nseg;
  return dtype == DGFX_F32 ? launch<float>(p, true, stream) : launch<__nv_bfloat16>(p, true, stream);
}

extern "C" int dgfx_gated_scan_step(const void* d_x, const void* d_gate, int dtype, int64_t n, int64_t channels,
                                    const float* d_state, void* d_h, float* d_new_state, dgfx_stream stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  DGFX_TRY(check_shape("dgfx_gated_scan_step", n, channels, 0, dtype));
  if (n == 0) return DGFX_OK;
  if (d_x == nullptr || d_gate == nullptr || d_state == nullptr || d_h == nullptr || d_new_state == nullptr) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_scan_step: null operand");
  }
  if (!quad_aligned(d_x, dtype) || !quad_aligned(d_gate, dtype) || !quad_aligned(d_h, dtype) ||
      !quad_aligned(d_state, DGFX_F32) || !quad_aligned(d_new_state, DGFX_F32)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_scan_step: operands must be aligned to 4 elements");
  }
  const int64_t quads = n * (channels / kCh);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(ceil_div(quads, 256), 148 * 32));
  if (dtype == DGFX_F32) {
    scan_step_kernel<float><<<grid, 256, 0, stream>>>(static_cast<const uint4*>(d_x), static_cast<const uint4*>(d_gate),
                                                      reinterpret_cast<const float4*>(d_state), quads,
                                                      static_cast<uint4*>(d_h), reinterpret_cast<float4*>(d_new_state));
  } else {
    scan_step_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(
        static_cast<const uint2*>(d_x), static_cast<const uint2*>(d_gate), reinterpret_cast<const float4*>(d_state),
        quads, static_cast<uint2*>(d_h), reinterpret_cast<float4*>(d_new_state));
  }
  DGFX_CUDA_TRY(cudaGetLastError());
  return DGFX_OK;
}
