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
// so windows of any lengths balance. The rows are cut into tiles of equal
// height; a tile's effect on the state that enters it is (A, H): state ->
// A state + H, and A < 0 marks a tile (or a part of one) that holds a
// restart, whose outgoing state is H alone (selected, not multiplied: a NaN
// of one window never reaches the next).
//
// One pass over the data, bound by HBM: persistent CTAs take tiles in order
// from a counter, each thread's inputs (kCh channels of a few consecutive
// rows) come by cp.async into its own slots of shared memory and move to registers,
// and the slots are refilled with the next tile's rows while this one's scan
// runs. A tile publishes its (A, H) as soon as it has them. The state that
// enters it is then composed from its predecessors' back to the tile where
// its first row's segment began, no further: from the (A, H) of the tiles of its
// group (32 tiles), of the groups of its supergroup (32 groups, each composed
// by its last tile) and the state that left the supergroup before; so a
// long segment costs a chain of one hop per 1024 tiles, and short windows
// look one tile back. The shape of that composition is fixed by the tile's
// number, so results do not change from run to run. A tile only waits for
// tiles taken before it; waits are bounded, and one that runs out is latched
// in the status word of dgfx_dense_check and ends all others.
//
// The backward pass runs the tiles from the last to the first. It computes
// the forward states again, from the state that entered the tile (saved by
// the forward pass: 4 bytes per tile and channel), instead of reading h.
//
// States, products and gradients of states are fp32; h, dx and dgate are
// rounded once when written. Rows outside [off[0], off[nseg]) are written as
// zeros and their inputs are never used.
#include <algorithm>
#include <string>

#include "layer_math.cuh"
#include "tensor_core.cuh"

namespace dgfx {
namespace {

constexpr int kThreads = 256;
constexpr int kCh = 4;  // channels per thread: 16 bytes of fp32, 8 of bf16
constexpr int kGroup = 32;
constexpr int kSuper = kGroup * kGroup;
constexpr int kSms = 148;

// Rows per thread: 64 bytes of each input.
template <class T>
constexpr int kRows = sizeof(T) == 2 ? 8 : 4;

// a = sigmoid(g) and 1 - a, both to full relative precision: e^-|g| never
// overflows, and neither comes from a subtraction.
__device__ __forceinline__ void gate_pair(float g, float* a, float* keep) {
  const float e = __expf(-fabsf(g));
  const float big = __fdividef(1.0f, 1.0f + e), small = e * big;
  *a = g >= 0.0f ? big : small;
  *keep = g >= 0.0f ? small : big;
}

// Shape of the tiling. Columns are groups of kCh channels; a tile is `width`
// columns wide (at most 16: 128 bytes of a bf16 row) and `subs` threads high.
struct Geometry {
  int32_t cols, width, across, subs, tile_rows;
  int64_t tiles;
};

Geometry geometry(int64_t rows, int64_t channels, int dtype) {
  Geometry g;
  g.cols = static_cast<int32_t>(channels / kCh);
  g.across = (g.cols + 15) / 16;
  g.width = (g.cols + g.across - 1) / g.across;
  g.subs = kThreads / g.width;
  g.tile_rows = g.subs * (dtype == DGFX_F32 ? kRows<float> : kRows<__nv_bfloat16>);
  g.tiles = ceil_div(std::max<int64_t>(rows, 1), g.tile_rows);
  return g;
}

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
  float* save;         // forward: state entering each tile [tiles, channels], or null
  const float* saved;  // backward: the same
  float2* tile_ah;     // [tiles, channels], by the order of processing
  float2* group_ah;    // [groups, channels]
  float* super_state;  // [supergroups, channels]
  uint32_t* tile_flag;  // [tiles, across]; then groups, supergroups, the counter and the abort word
  uint32_t* group_flag;
  uint32_t* super_flag;
  uint32_t* counter;
  uint32_t* aborted;
  int32_t* first_seg;  // per tile: the segment of its first row (or the next one)
  int32_t* origin;     // per tile: the tile (by number) where the segment that enters it began
  unsigned int* err;
  int64_t rows, channels, nseg;
  int64_t clear_words;
  Geometry geo;
  int32_t up;  // backward: tiles are processed from the last to the first
};

// ---------------------------------------------------------------------------
// Before the scan: where every tile stands among the segments, outputs of the
// segments without rows, and cleared flags. A warp per segment.
// ---------------------------------------------------------------------------
__global__ void scan_plan_kernel(Params p, const float* __restrict__ empty_in, float* __restrict__ empty_out) {
  const int64_t threads = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int lane = threadIdx.x & 31;
  for (int64_t i = t; i < p.clear_words; i += threads) p.tile_flag[i] = 0;
  const int64_t lo = clamp64(p.off[0], 0, p.rows), hi = clamp64(p.off[p.nseg], lo, p.rows);
  const int64_t tr = p.geo.tile_rows;
  // Tiles whose first row (last row, going up) lies outside of every segment
  // have nothing to wait for.
  for (int64_t i = t; i < p.geo.tiles; i += threads) {
    const int64_t row0 = i * tr, row1 = (row0 + tr < p.rows ? row0 + tr : p.rows) - 1;
    if (row0 < lo || row0 >= hi) p.first_seg[i] = row0 < lo ? 0 : static_cast<int32_t>(p.nseg);
    const int64_t edge = p.up ? row1 : row0;
    if (edge < lo || edge >= hi) p.origin[i] = static_cast<int32_t>(i);
  }
  for (int64_t s = t >> 5; s < p.nseg; s += threads >> 5) {
    const int64_t b = clamp64(p.off[s], lo, hi), e = clamp64(p.off[s + 1], b, hi);
    if (b == e) {
      if (empty_out != nullptr) {
        for (int64_t c = lane; c < p.channels; c += 32) {
          empty_out[s * p.channels + c] = empty_in != nullptr ? empty_in[s * p.channels + c] : 0.0f;
        }
      }
      continue;
    }
    // Tiles whose first row lies in [b, e).
    for (int64_t i = (b + tr - 1) / tr + lane; i * tr < e; i += 32) {
      p.first_seg[i] = static_cast<int32_t>(s);
      if (!p.up) p.origin[i] = static_cast<int32_t>(b / tr);
    }
    if (p.up) {  // tiles whose last row does
      for (int64_t i = b / tr + lane; i < p.geo.tiles; i += 32) {
        const int64_t row1 = (i * tr + tr < p.rows ? i * tr + tr : p.rows) - 1;
        if (row1 >= e) break;
        p.origin[i] = static_cast<int32_t>((e - 1) / tr);
      }
    }
  }
}

// The segment structure of one tile: for each row the segment that starts
// (ends) there, -1 if none. [lo, hi) are the rows inside any segment.
struct TileSegments {
  int32_t* starts;
  int32_t* ends;
  int64_t lo, hi;
};

__device__ __forceinline__ void find_segments(const Params& p, int64_t tile, TileSegments& ts) {
  const int64_t row0 = tile * p.geo.tile_rows;
  const int64_t row_end = row0 + p.geo.tile_rows < p.rows ? row0 + p.geo.tile_rows : p.rows;
  // Clamped: offsets that do not ascend may leave it unset.
  const int64_t first = clamp64(__ldcg(p.first_seg + tile), 0, p.nseg);
  for (int i = threadIdx.x; i < p.geo.tile_rows; i += kThreads) {
    ts.starts[i] = -1;
    ts.ends[i] = -1;
  }
  __syncthreads();
  for (int64_t s = first + threadIdx.x;; s += kThreads) {
    bool more = false;
    if (s < p.nseg) {
      const int64_t b = __ldg(p.off + s), e = __ldg(p.off + s + 1);
      if (b < e) {
        if (b >= row0 && b < row_end) ts.starts[b - row0] = static_cast<int32_t>(s);
        if (e > row0 && e <= row_end) ts.ends[e - 1 - row0] = static_cast<int32_t>(s);
      }
      more = threadIdx.x == kThreads - 1 && b < row_end;
    }
    if (!__syncthreads_or(more)) break;
  }
}

__device__ __forceinline__ float enter(float a, float h, float state) { return a < 0.0f ? h : fmaf(a, state, h); }

// (a, h) followed by (na, nh).
__device__ __forceinline__ void then(float* a, float* h, float na, float nh) {
  *h = enter(na, nh, *h);
  *a = (na < 0.0f || *a < 0.0f) ? -1.0f : *a * na;
}

// Exclusive composition of the subs' (A, H) in place, `up` from the last row
// to the first; the tile's own (A, H) in *ta, *th. One thread per channel.
__device__ __forceinline__ void compose(float* sa, float* sh, int chans, int subs, bool up, int ch, float* ta,
                                        float* th) {
  float a = 1.0f, h = 0.0f;
  for (int k = 0; k < subs; ++k) {
    const int i = (up ? subs - 1 - k : k) * chans + ch;
    const float ca = sa[i], chv = sh[i];
    sa[i] = a;
    sh[i] = h;
    then(&a, &h, ca, chv);
  }
  *ta = a;
  *th = h;
}

__device__ __forceinline__ uint32_t load_flag(const uint32_t* f) {
  uint32_t v;
  asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(f) : "memory");
  return v;
}

__device__ __forceinline__ void raise_flag(uint32_t* f) {
  asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(f), "r"(1u) : "memory");
}

// Waits (one warp) until every lane's flag is up; lanes without one pass
// null. Gives up after 2 s, or when another wait of this launch did.
__device__ __forceinline__ void wait_flags(const Params& p, const uint32_t* flag) {
  const uint64_t t0 = now_ns();
  for (uint32_t i = 1;; ++i) {
    const bool up = flag == nullptr || load_flag(flag) != 0;
    if (__all_sync(0xffffffffu, up)) return;
    if ((i & 63u) == 0) {
      bool stop = false;
      if ((threadIdx.x & 31) == 0) {
        stop = load_flag(p.aborted) != 0;
        if (!stop && now_ns() - t0 > kWaitNs) {
          raise_flag(p.aborted);
          atomicOr(p.err, 2u);
          stop = true;
        }
      }
      if (__any_sync(0xffffffffu, stop)) return;
    }
  }
}

// Work of one CTA on one tile in the order of processing: publishing and the
// state that enters. fold: (A, H) of consecutive tiles or groups, composed by
// all threads (each a contiguous part per channel, then the parts in order).
struct Chain {
  const Params& p;
  float2* parts;  // [kThreads]
  float* state;   // [chans]: the state that enters the tile
  int chans, part, lanes, my_ch, my_part;
  int64_t gch;  // this thread's channel of the fold

  __device__ Chain(const Params& params, float2* parts_, float* state_, int part_)
      : p(params), parts(parts_), state(state_), chans(params.geo.width * kCh), part(part_) {
    lanes = kThreads / chans;
    my_part = threadIdx.x / chans;
    my_ch = threadIdx.x - my_part * chans;
    gch = static_cast<int64_t>(part) * chans + my_ch;
  }

  // Composes groups [g0, g1) and then tiles [t0, t1) for this thread's
  // channel; valid in the threads of part 0. Contains barriers.
  __device__ float2 fold(int64_t g0, int64_t g1, int64_t t0, int64_t t1) {
    const int ng = static_cast<int>(g1 - g0), n = ng + static_cast<int>(t1 - t0);
    const int each = (n + lanes - 1) / lanes;
    float a = 1.0f, h = 0.0f;
    if (my_part < lanes && gch < p.channels) {
      const int from = my_part * each, to = min(n, from + each);
#pragma unroll 4
      for (int i = from; i < to; ++i) {
        const float2* src = i < ng ? p.group_ah + (g0 + i) * p.channels : p.tile_ah + (t0 + i - ng) * p.channels;
        const float2 v = __ldcg(src + gch);
        then(&a, &h, v.x, v.y);
      }
    }
    parts[threadIdx.x] = make_float2(a, h);
    __syncthreads();
    a = 1.0f;
    h = 0.0f;
    if (my_part == 0) {
      for (int k = 0; k < lanes; ++k) {
        const float2 v = parts[k * chans + my_ch];
        then(&a, &h, v.x, v.y);
      }
    }
    __syncthreads();
    return make_float2(a, h);
  }

  // Publishes tile j's (A, H) (threads of part 0 hold it) and its group's, if
  // j is the last of it.
  __device__ void publish(int64_t j, float2 ah) {
    if (my_part == 0 && gch < p.channels) __stcg(p.tile_ah + j * p.channels + gch, ah);
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) raise_flag(p.tile_flag + j * p.geo.across + part);
    if (j % kGroup != kGroup - 1) return;
    const int64_t t0 = j - (kGroup - 1);
    if (threadIdx.x < 32) wait_flags(p, p.tile_flag + (t0 + threadIdx.x) * p.geo.across + part);
    __syncthreads();
    const float2 g = fold(0, 0, t0, j + 1);
    if (my_part == 0 && gch < p.channels) __stcg(p.group_ah + j / kGroup * p.channels + gch, g);
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) raise_flag(p.group_flag + j / kGroup * p.geo.across + part);
  }

  // The state that enters tile j, whose segment began in tile k0 <= j (all in the
  // order of processing), into state[]; `ah` is the tile's own (part 0).
  // Publishes the state that leaves j if it ends a supergroup.
  __device__ void enter_tile(int64_t j, int64_t k0, float2 ah) {
    float st = 0.0f;
    if (k0 < j) {
      const int64_t gs = j / kGroup * kGroup, ss = j / kSuper * kSuper;
      const int64_t t0 = k0 > gs ? k0 : gs;
      const int64_t g1 = gs / kGroup;
      int64_t g0 = g1;
      if (k0 < gs) g0 = k0 > ss ? k0 / kGroup : ss / kGroup;
      const bool super = k0 < ss;
      if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        wait_flags(p, t0 + lane < j ? p.tile_flag + (t0 + lane) * p.geo.across + part : nullptr);
        if (g0 < g1) wait_flags(p, g0 + lane < g1 ? p.group_flag + (g0 + lane) * p.geo.across + part : nullptr);
        if (super) wait_flags(p, lane == 0 ? p.super_flag + (ss / kSuper - 1) * p.geo.across + part : nullptr);
      }
      __syncthreads();
      const float2 f = fold(g0, g1, t0, j);
      if (my_part == 0 && gch < p.channels) {
        if (super) st = __ldcg(p.super_state + (ss / kSuper - 1) * p.channels + gch);
        st = enter(f.x, f.y, st);
      }
    }
    if (my_part == 0) state[my_ch] = st;
    if (j % kSuper == kSuper - 1) {
      if (my_part == 0 && gch < p.channels) {
        __stcg(p.super_state + j / kSuper * p.channels + gch, enter(ah.x, ah.y, st));
      }
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) raise_flag(p.super_flag + j / kSuper * p.geo.across + part);
    }
    __syncthreads();
  }
};

// One quad to this thread's slot; zeros instead if it is not there.
template <class T>
__device__ __forceinline__ void fetch(void* slot, const void* src, bool there) {
  constexpr int kBytes = sizeof(typename Quad<T>::raw);
  const int n = there ? kBytes : 0;
  if (kBytes == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(slot)), "l"(src), "r"(n) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(slot)), "l"(src), "r"(n) : "memory");
  }
}

__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void fetch_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared memory of a CTA: INPUTS x rows x threads slots of quads, the subs'
// (A, H), the fold's parts, the entering state, the tile's segments.
template <class T, int INPUTS, bool KEEP>
struct Smem {
  using raw = typename Quad<T>::raw;
  raw* slots;
  float4* keep;  // backward: 1 - a of this thread's rows
  float *sa, *sh, *state;
  float2* parts;
  int32_t *starts, *ends;
  static size_t bytes(const Geometry& g) {
    return static_cast<size_t>(INPUTS) * kRows<T> * kThreads * sizeof(raw) +
           (KEEP ? static_cast<size_t>(kRows<T>) * kThreads * sizeof(float4) : 0) +
           2 * kThreads * kCh * sizeof(float) + kThreads * sizeof(float2) + 64 * sizeof(float) +
           2 * static_cast<size_t>(g.tile_rows) * sizeof(int32_t);
  }
  __device__ Smem(void* base, const Geometry& g) {
    char* b = static_cast<char*>(base);
    auto take = [&](size_t n) {
      char* r = b;
      b += n;
      return r;
    };
    slots = reinterpret_cast<raw*>(take(static_cast<size_t>(INPUTS) * kRows<T> * kThreads * sizeof(raw)));
    keep = reinterpret_cast<float4*>(take(KEEP ? kRows<T> * kThreads * sizeof(float4) : 0));
    sa = reinterpret_cast<float*>(take(kThreads * kCh * sizeof(float)));
    sh = reinterpret_cast<float*>(take(kThreads * kCh * sizeof(float)));
    parts = reinterpret_cast<float2*>(take(kThreads * sizeof(float2)));
    state = reinterpret_cast<float*>(take(64 * sizeof(float)));
    starts = reinterpret_cast<int32_t*>(take(g.tile_rows * sizeof(int32_t)));
    ends = reinterpret_cast<int32_t*>(take(g.tile_rows * sizeof(int32_t)));
  }
  __device__ raw* slot(int input, int i) { return slots + (input * kRows<T> + i) * kThreads + threadIdx.x; }
};

// Where a ticket's tile lies and this thread in it.
struct Spot {
  int64_t j, tile, r0;  // order of processing, number, this thread's first row
  int part, col;
  bool on;
};

__device__ __forceinline__ Spot spot_of(const Params& p, uint32_t ticket, int sub, int lc, int rows_each) {
  Spot s;
  s.j = ticket / p.geo.across;
  s.part = static_cast<int>(ticket - s.j * p.geo.across);
  s.tile = p.up ? p.geo.tiles - 1 - s.j : s.j;
  s.col = s.part * p.geo.width + lc;
  s.on = sub < p.geo.subs && s.col < p.geo.cols;
  s.r0 = s.tile * p.geo.tile_rows + static_cast<int64_t>(sub) * rows_each;
  return s;
}

template <class T, int N>
__device__ __forceinline__ void fetch_rows(const Params& p, const Spot& s, const void* base, Smem<T, N, N == 3>& sm,
                                           int input) {
  using raw = typename Quad<T>::raw;
  const raw* src = static_cast<const raw*>(base);
#pragma unroll
  for (int i = 0; i < kRows<T>; ++i) {
    const bool there = s.on && s.r0 + i < p.rows && src != nullptr;
    fetch<T>(sm.slot(input, i), there ? src + (s.r0 + i) * p.geo.cols + s.col : static_cast<const raw*>(p.x), there);
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads, 2) scan_forward_kernel(Params p) {
  using Q = Quad<T>;
  constexpr int R = kRows<T>;
  extern __shared__ __align__(16) char smem_raw[];
  __shared__ uint32_t next_ticket;
  Smem<T, 2, false> sm(smem_raw, p.geo);
  const int sub = threadIdx.x / p.geo.width, lc = threadIdx.x - sub * p.geo.width;
  const int chans = p.geo.width * kCh, slot = sub * chans + lc * kCh;
  const uint32_t tickets = static_cast<uint32_t>(p.geo.tiles * p.geo.across);
  TileSegments ts;
  ts.starts = sm.starts;
  ts.ends = sm.ends;
  ts.lo = clamp64(p.off[0], 0, p.rows);
  ts.hi = clamp64(p.off[p.nseg], ts.lo, p.rows);

  if (threadIdx.x == 0) next_ticket = atomicAdd(p.counter, 1u);
  __syncthreads();
  uint32_t ticket = next_ticket;
  Spot s = spot_of(p, ticket, sub, lc, R);
  if (ticket < tickets) {
    fetch_rows<T, 2>(p, s, p.gate, sm, 0);
    fetch_rows<T, 2>(p, s, p.x, sm, 1);
  }
  fetch_commit();
  while (ticket < tickets) {
    __syncthreads();  // everyone has read next_ticket
    if (threadIdx.x == 0) next_ticket = atomicAdd(p.counter, 1u);
    find_segments(p, s.tile, ts);
    const uint32_t ahead = next_ticket;
    const int64_t origin = clamp64(__ldcg(p.origin + s.tile), 0, s.tile);
    fetch_wait<0>();

    float a[R][kCh], u[R][kCh];
    float pa[kCh], ph[kCh];
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      pa[c] = 1.0f;
      ph[c] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float xv[kCh], gv[kCh];
      Q::unpack(*sm.slot(0, i), gv);
      Q::unpack(*sm.slot(1, i), xv);
      const bool inside = s.r0 + i >= ts.lo && s.r0 + i < ts.hi;
      const int32_t seg = s.on ? ts.starts[sub * R + i] : -1;
      const bool restart = seg >= 0 || !inside;
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        float av, keep;
        gate_pair(gv[c], &av, &keep);
        float uv = keep * xv[c];
        if (seg >= 0 && p.initial != nullptr) uv = fmaf(av, __ldg(p.initial + seg * p.channels + s.col * kCh + c), uv);
        a[i][c] = restart ? -1.0f : av;
        u[i][c] = inside ? uv : 0.0f;
        ph[c] = restart ? u[i][c] : fmaf(av, ph[c], uv);
        pa[c] = (restart || pa[c] < 0.0f) ? -1.0f : pa[c] * av;
      }
    }
    // The next tile's rows into the slots just read.
    const Spot ns = spot_of(p, ahead, sub, lc, R);
    if (ahead < tickets) {
      fetch_rows<T, 2>(p, ns, p.gate, sm, 0);
      fetch_rows<T, 2>(p, ns, p.x, sm, 1);
    }
    fetch_commit();
    if (sub < p.geo.subs) {
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        sm.sa[slot + c] = pa[c];
        sm.sh[slot + c] = ph[c];
      }
    }
    __syncthreads();
    Chain chain(p, sm.parts, sm.state, s.part);
    float2 ah = make_float2(1.0f, 0.0f);
    if (threadIdx.x < chans) compose(sm.sa, sm.sh, chans, p.geo.subs, false, threadIdx.x, &ah.x, &ah.y);
    chain.publish(s.j, ah);
    chain.enter_tile(s.j, origin, ah);
    if (p.save != nullptr && threadIdx.x < chans && chain.gch < p.channels) {
      p.save[s.tile * p.channels + chain.gch] = sm.state[threadIdx.x];
    }
    if (s.on) {
      float st[kCh];
#pragma unroll
      for (int c = 0; c < kCh; ++c) st[c] = enter(sm.sa[slot + c], sm.sh[slot + c], sm.state[lc * kCh + c]);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (s.r0 + i < p.rows) {
#pragma unroll
          for (int c = 0; c < kCh; ++c) st[c] = enter(a[i][c], u[i][c], st[c]);
          if (p.h != nullptr) static_cast<typename Q::raw*>(p.h)[(s.r0 + i) * p.geo.cols + s.col] = Q::pack(st);
          const int32_t seg = ts.ends[sub * R + i];
          if (seg >= 0 && p.final != nullptr) {
            *reinterpret_cast<float4*>(p.final + seg * p.channels + s.col * kCh) = make_float4(st[0], st[1], st[2], st[3]);
          }
        }
      }
    }
    ticket = ahead;
    s = ns;
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads, 2) scan_backward_kernel(Params p) {
  using Q = Quad<T>;
  constexpr int R = kRows<T>;
  extern __shared__ __align__(16) char smem_raw[];
  __shared__ uint32_t next_ticket;
  Smem<T, 3, true> sm(smem_raw, p.geo);
  const int sub = threadIdx.x / p.geo.width, lc = threadIdx.x - sub * p.geo.width;
  const int chans = p.geo.width * kCh, slot = sub * chans + lc * kCh;
  const uint32_t tickets = static_cast<uint32_t>(p.geo.tiles * p.geo.across);
  TileSegments ts;
  ts.starts = sm.starts;
  ts.ends = sm.ends;
  ts.lo = clamp64(p.off[0], 0, p.rows);
  ts.hi = clamp64(p.off[p.nseg], ts.lo, p.rows);

  if (threadIdx.x == 0) next_ticket = atomicAdd(p.counter, 1u);
  __syncthreads();
  uint32_t ticket = next_ticket;
  Spot s = spot_of(p, ticket, sub, lc, R);
  if (ticket < tickets) {
    fetch_rows<T, 3>(p, s, p.gate, sm, 0);
    fetch_rows<T, 3>(p, s, p.x, sm, 1);
  }
  fetch_commit();
  if (ticket < tickets) fetch_rows<T, 3>(p, s, p.grad, sm, 2);
  fetch_commit();
  while (ticket < tickets) {
    __syncthreads();
    if (threadIdx.x == 0) next_ticket = atomicAdd(p.counter, 1u);
    find_segments(p, s.tile, ts);
    const uint32_t ahead = next_ticket;
    const Spot ns = spot_of(p, ahead, sub, lc, R);
    const int64_t origin = clamp64(__ldcg(p.origin + s.tile), s.tile, p.geo.tiles - 1);
    fetch_wait<1>();  // gate and x are here, grad may still be on its way

    // The forward states of this tile again.
    float a[R][kCh], q[R][kCh];
    float pa[kCh], ph[kCh];
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      pa[c] = 1.0f;
      ph[c] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float xv[kCh], gv[kCh], kv[kCh];
      Q::unpack(*sm.slot(0, i), gv);
      Q::unpack(*sm.slot(1, i), xv);
      const bool inside = s.r0 + i >= ts.lo && s.r0 + i < ts.hi;
      const int32_t seg = s.on ? ts.starts[sub * R + i] : -1;
      const bool restart = seg >= 0 || !inside;
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        gate_pair(gv[c], &a[i][c], &kv[c]);
        float uv = kv[c] * xv[c];
        if (seg >= 0 && p.initial != nullptr) {
          uv = fmaf(a[i][c], __ldg(p.initial + seg * p.channels + s.col * kCh + c), uv);
        }
        ph[c] = restart ? (inside ? uv : 0.0f) : fmaf(a[i][c], ph[c], uv);
        pa[c] = (restart || pa[c] < 0.0f) ? -1.0f : pa[c] * a[i][c];
      }
      sm.keep[i * kThreads + threadIdx.x] = make_float4(kv[0], kv[1], kv[2], kv[3]);
    }
    if (sub < p.geo.subs) {
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        sm.sa[slot + c] = pa[c];
        sm.sh[slot + c] = ph[c];
      }
    }
    __syncthreads();
    float2 ah = make_float2(1.0f, 0.0f);
    if (threadIdx.x < chans) compose(sm.sa, sm.sh, chans, p.geo.subs, false, threadIdx.x, &ah.x, &ah.y);
    __syncthreads();
    float st[kCh];
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      st[c] = s.on ? enter(sm.sa[slot + c], sm.sh[slot + c], __ldg(p.saved + s.tile * p.channels + s.col * kCh + c))
                   : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float xv[kCh];
      Q::unpack(*sm.slot(1, i), xv);
      const float4 k4 = sm.keep[i * kThreads + threadIdx.x];
      const float kv[kCh] = {k4.x, k4.y, k4.z, k4.w};
      const int32_t seg = s.on ? ts.starts[sub * R + i] : -1;
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        if (seg >= 0) st[c] = p.initial != nullptr ? __ldg(p.initial + seg * p.channels + s.col * kCh + c) : 0.0f;
        q[i][c] = (st[c] - xv[c]) * (a[i][c] * kv[c]);
        st[c] = fmaf(a[i][c], st[c], kv[c] * xv[c]);
      }
    }
    if (ahead < tickets) {  // gate and x of the next tile into the slots just read
      fetch_rows<T, 3>(p, ns, p.gate, sm, 0);
      fetch_rows<T, 3>(p, ns, p.x, sm, 1);
    }
    fetch_commit();
    fetch_wait<1>();  // grad of this tile

    // e_t = a_t (d_t + e_{t+1}) from the last row of the thread to its first.
    float pe[kCh];
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      pa[c] = 1.0f;
      pe[c] = 0.0f;
    }
#pragma unroll
    for (int i = R - 1; i >= 0; --i) {
      float dv[kCh];
      Q::unpack(*sm.slot(2, i), dv);
      const int32_t seg = s.on ? ts.ends[sub * R + i] : -1;
      const bool inside = s.r0 + i >= ts.lo && s.r0 + i < ts.hi;
      const bool restart = seg >= 0 || !inside;
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        if (seg >= 0 && p.grad_final != nullptr) dv[c] += __ldg(p.grad_final + seg * p.channels + s.col * kCh + c);
        pe[c] = inside ? a[i][c] * (restart ? dv[c] : dv[c] + pe[c]) : 0.0f;
        pa[c] = (restart || pa[c] < 0.0f) ? -1.0f : pa[c] * a[i][c];
      }
    }
    __syncthreads();  // the forward composition has been read
    if (sub < p.geo.subs) {
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        sm.sa[slot + c] = pa[c];
        sm.sh[slot + c] = pe[c];
      }
    }
    __syncthreads();
    Chain chain(p, sm.parts, sm.state, s.part);
    ah = make_float2(1.0f, 0.0f);
    if (threadIdx.x < chans) compose(sm.sa, sm.sh, chans, p.geo.subs, true, threadIdx.x, &ah.x, &ah.y);
    chain.publish(s.j, ah);
    chain.enter_tile(s.j, p.geo.tiles - 1 - origin, ah);
    if (s.on) {
      float e[kCh];
#pragma unroll
      for (int c = 0; c < kCh; ++c) e[c] = enter(sm.sa[slot + c], sm.sh[slot + c], sm.state[lc * kCh + c]);
#pragma unroll
      for (int i = R - 1; i >= 0; --i) {
        if (s.r0 + i < p.rows) {
          const bool inside = s.r0 + i >= ts.lo && s.r0 + i < ts.hi;
          const int32_t end = ts.ends[sub * R + i], seg = ts.starts[sub * R + i];
          const float4 k4 = sm.keep[i * kThreads + threadIdx.x];
          const float kv[kCh] = {k4.x, k4.y, k4.z, k4.w};
          float dv[kCh], dx[kCh], dg[kCh];
          Q::unpack(*sm.slot(2, i), dv);
#pragma unroll
          for (int c = 0; c < kCh; ++c) {
            if (end >= 0) e[c] = p.grad_final != nullptr ? __ldg(p.grad_final + end * p.channels + s.col * kCh + c) : 0.0f;
            const float delta = dv[c] + e[c];
            e[c] = inside ? a[i][c] * delta : 0.0f;
            dx[c] = inside ? kv[c] * delta : 0.0f;
            dg[c] = inside ? delta * q[i][c] : 0.0f;
          }
          static_cast<typename Q::raw*>(p.dx)[(s.r0 + i) * p.geo.cols + s.col] = Q::pack(dx);
          static_cast<typename Q::raw*>(p.dgate)[(s.r0 + i) * p.geo.cols + s.col] = Q::pack(dg);
          if (seg >= 0 && p.dinitial != nullptr) {
            *reinterpret_cast<float4*>(p.dinitial + seg * p.channels + s.col * kCh) = make_float4(e[0], e[1], e[2], e[3]);
          }
        }
      }
    }
    if (ahead < tickets) fetch_rows<T, 3>(p, ns, p.grad, sm, 2);
    fetch_commit();
    ticket = ahead;
    s = ns;
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
  if (channels > (int64_t(1) << 20) || nseg >= (int64_t(1) << 31) || rows > (int64_t(1) << 40) ||
      geometry(rows, channels, dtype).tiles * geometry(rows, channels, dtype).across >= (int64_t(1) << 31)) {
    return fail(DGFX_ERR_UNSUPPORTED, std::string(who) + ": sizes out of range");
  }
  return DGFX_OK;
}

// Quads are loaded whole, fp32 states as 16-byte vectors.
bool quad_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == DGFX_F32 ? 15u : 7u)) == 0;
}

size_t carve(void* base, size_t cap, const Geometry& g, int64_t channels, Params* p, bool* ok) {
  Arena arena(base, cap);
  const int64_t groups = ceil_div(g.tiles, kGroup), supers = ceil_div(g.tiles, kSuper);
  p->tile_ah = arena.take<float2>(static_cast<size_t>(g.tiles) * channels);
  p->group_ah = arena.take<float2>(static_cast<size_t>(groups) * channels);
  p->super_state = arena.take<float>(static_cast<size_t>(supers) * channels);
  p->clear_words = (g.tiles + groups + supers) * g.across + 2;
  p->tile_flag = arena.take<uint32_t>(static_cast<size_t>(p->clear_words));
  p->first_seg = arena.take<int32_t>(static_cast<size_t>(g.tiles));
  p->origin = arena.take<int32_t>(static_cast<size_t>(g.tiles));
  if (base != nullptr) {
    p->group_flag = p->tile_flag + g.tiles * g.across;
    p->super_flag = p->group_flag + groups * g.across;
    p->counter = p->super_flag + supers * g.across;
    p->aborted = p->counter + 1;
  }
  *ok = arena.ok();
  return arena.used;
}

unsigned plan_grid(const Params& p) {
  const int64_t items = std::max(std::max(p.clear_words, p.geo.tiles), p.nseg * 32);
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(ceil_div(items, 256), kSms * 8)));
}

template <class T, bool BACKWARD>
int launch(const Params& p, cudaStream_t stream) {
  auto kernel = BACKWARD ? scan_backward_kernel<T> : scan_forward_kernel<T>;
  const size_t smem = BACKWARD ? Smem<T, 3, true>::bytes(p.geo) : Smem<T, 2, false>::bytes(p.geo);
  if (smem > 48 * 1024) {
    static std::once_flag once[64];
    int dev = 0;
    DGFX_CUDA_TRY(cudaGetDevice(&dev));
    cudaError_t err = cudaSuccess;
    std::call_once(once[dev & 63], [&]() {
      err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 112 * 1024);
    });
    DGFX_CUDA_TRY(err);
  }
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(p.geo.tiles * p.geo.across, 2 * kSms));
  kernel<<<grid, kThreads, smem, stream>>>(p);
  DGFX_CUDA_TRY(cudaGetLastError());
  return DGFX_OK;
}

}  // namespace
}  // namespace dgfx

using namespace dgfx;

extern "C" int dgfx_gated_scan_workspace_size(int64_t rows, int64_t channels, int dtype, size_t* workspace_bytes,
                                              size_t* saved_bytes) {
  DGFX_TRY(check_shape("dgfx_gated_scan_workspace_size", rows, channels, 0, dtype));
  const Geometry g = geometry(rows, channels, dtype);
  Params p{};
  bool ok;
  if (workspace_bytes != nullptr) *workspace_bytes = carve(nullptr, 0, g, channels, &p, &ok);
  if (saved_bytes != nullptr) *saved_bytes = static_cast<size_t>(g.tiles) * channels * sizeof(float);
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
      !quad_aligned(d_final, DGFX_F32)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_scan: operands must be aligned to 4 elements");
  }
  Params p{};
  p.geo = geometry(rows, channels, dtype);
  bool ok = false;
  carve(d_workspace, workspace_bytes, p.geo, channels, &p, &ok);
  if (d_workspace == nullptr || !ok) return fail(DGFX_ERR_WORKSPACE, "dgfx_gated_scan: workspace too small");
  p.err = dense_err_word();
  if (p.err == nullptr) return fail(DGFX_ERR_CUDA, "dgfx_gated_scan: status word unavailable");
  p.x = d_x;
  p.gate = d_gate;
  p.off = d_offsets;
  p.initial = d_initial;
  p.h = d_h;
  p.final = d_final;
  p.save = d_saved;
  p.rows = rows;
  p.channels = channels;
  p.nseg = nseg;
  scan_plan_kernel<<<plan_grid(p), 256, 0, stream>>>(p, d_initial, d_final);
  DGFX_CUDA_TRY(cudaGetLastError());
  if (rows == 0) return DGFX_OK;
  return dtype == DGFX_F32 ? launch<float, false>(p, stream) : launch<__nv_bfloat16, false>(p, stream);
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
      !quad_aligned(d_dx, dtype) || !quad_aligned(d_dgate, dtype) || !quad_aligned(d_dinitial, DGFX_F32)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_scan_backward: operands must be aligned to 4 elements");
  }
  Params p{};
  p.geo = geometry(rows, channels, dtype);
  bool ok = false;
  carve(d_workspace, workspace_bytes, p.geo, channels, &p, &ok);
  if (d_workspace == nullptr || !ok) return fail(DGFX_ERR_WORKSPACE, "dgfx_gated_scan_backward: workspace too small");
  p.err = dense_err_word();
  if (p.err == nullptr) return fail(DGFX_ERR_CUDA, "dgfx_gated_scan_backward: status word unavailable");
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
  p.rows = rows;
  p.channels = channels;
  p.nseg = nseg;
  p.up = 1;
  scan_plan_kernel<<<plan_grid(p), 256, 0, stream>>>(p, d_grad_final, d_dinitial);
  DGFX_CUDA_TRY(cudaGetLastError());
  if (rows == 0) return DGFX_OK;
  return dtype == DGFX_F32 ? launch<float, true>(p, stream) : launch<__nv_bfloat16, true>(p, stream);
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
