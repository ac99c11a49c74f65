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
// so windows of any lengths balance: the rows are cut into tiles of equal
// height, a tile's effect on the state that enters it is (A, H): state ->
// A state + H, and A < 0 marks a tile (or a part of one) that holds a
// restart, whose outgoing state is H alone (selected, not multiplied: a NaN
// of one window never reaches the next). A thread owns kCh adjacent channels of
// kRows consecutive rows; the threads of a tile stand side by side over the
// channels (coalesced rows) and one above the other over the rows. States, products and
// gradients of states are fp32; h, dx and dgate are rounded once when
// written. Rows outside [off[0], off[nseg]) are written as zeros and their
// inputs are never used.
#include <algorithm>
#include <string>

#include "layer_math.cuh"

namespace dgfx {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 8;  // rows per thread
constexpr int kCh = 4;    // channels per thread: 16 bytes of fp32, 8 of bf16
constexpr int kMaxTile = kThreads * kRows;

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

Geometry geometry(int64_t rows, int64_t channels) {
  Geometry g;
  g.cols = static_cast<int32_t>(channels / kCh);
  g.across = (g.cols + 15) / 16;
  g.width = (g.cols + g.across - 1) / g.across;
  g.subs = kThreads / g.width;
  g.tile_rows = g.subs * kRows;
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
  float* states;  // [tiles, channels]: state entering each tile (from above, or from below going backward)
  float* agg_a;   // [tiles, channels]
  float* agg_h;
  const float* saved;  // backward: the forward pass's states
  int64_t rows, channels, nseg;
  Geometry geo;
};

// The segment structure of one tile: for each row the segment that starts
// (ends) there, -1 if none. [lo, hi) are the rows inside any segment.
struct TileSegments {
  int32_t starts[kMaxTile];
  int32_t ends[kMaxTile];
  int64_t lo, hi, first;
};

__device__ __forceinline__ void find_segments(const Params& p, int64_t row0, int tile_rows, TileSegments& ts) {
  for (int i = threadIdx.x; i < tile_rows; i += kThreads) {
    ts.starts[i] = -1;
    ts.ends[i] = -1;
  }
  if (threadIdx.x < 32) {
    const int64_t first = warp_first_segment(p.off, p.nseg, row0);
    if (threadIdx.x == 0) {
      ts.first = first;
      ts.lo = clamp64(p.off[0], 0, p.rows);
      ts.hi = clamp64(p.off[p.nseg], ts.lo, p.rows);
    }
  }
  __syncthreads();
  const int64_t row_end = min(row0 + tile_rows, p.rows);
  for (int64_t s0 = ts.first; s0 < p.nseg; s0 += kThreads) {
    const int64_t s = s0 + threadIdx.x;
    if (s < p.nseg) {
      const int64_t b = p.off[s], e = p.off[s + 1];
      if (b < e) {
        if (b >= row0 && b < row_end) ts.starts[b - row0] = static_cast<int32_t>(s);
        if (e > row0 && e <= row_end) ts.ends[e - 1 - row0] = static_cast<int32_t>(s);
      }
    }
    if (p.off[s0] >= row_end) break;  // the same for every thread
  }
  __syncthreads();
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
    h = ca < 0.0f ? chv : fmaf(ca, h, chv);
    a = (ca < 0.0f || a < 0.0f) ? -1.0f : a * ca;
  }
  *ta = a;
  *th = h;
}

__device__ __forceinline__ float enter(float a, float h, float state) { return a < 0.0f ? h : fmaf(a, state, h); }

// kAggregate: write the tile's (A, H). kApply: take the state that enters
// the tile and write the outputs.
enum { kAggregate = 0, kApply = 1 };

template <class T, int PHASE>
__global__ void __launch_bounds__(kThreads, 2) scan_forward_kernel(Params p) {
  using Q = Quad<T>;
  __shared__ TileSegments ts;
  __shared__ float sa[kThreads * kCh], sh[kThreads * kCh];
  const int32_t tile = static_cast<int32_t>(blockIdx.x / p.geo.across), part = blockIdx.x % p.geo.across;
  const int sub = threadIdx.x / p.geo.width, lc = threadIdx.x - sub * p.geo.width;
  const int col = part * p.geo.width + lc;
  const bool on = sub < p.geo.subs && col < p.geo.cols;
  const int64_t row0 = static_cast<int64_t>(tile) * p.geo.tile_rows;
  const int64_t r0 = row0 + static_cast<int64_t>(sub) * kRows;
  const int chans = p.geo.width * kCh;
  const typename Q::raw* x = static_cast<const typename Q::raw*>(p.x);
  const typename Q::raw* gate = static_cast<const typename Q::raw*>(p.gate);

  typename Q::raw xr[kRows], gr[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const bool ok = on && r0 + i < p.rows;
    gr[i] = ok ? __ldg(gate + (r0 + i) * p.geo.cols + col) : Q::zero();
    xr[i] = ok ? __ldg(x + (r0 + i) * p.geo.cols + col) : Q::zero();
  }
  find_segments(p, row0, p.geo.tile_rows, ts);

  float a[kRows][kCh], u[kRows][kCh];
  float pa[kCh], ph[kCh];
#pragma unroll
  for (int c = 0; c < kCh; ++c) {
    pa[c] = 1.0f;
    ph[c] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    float xv[kCh], gv[kCh];
    Q::unpack(xr[i], xv);
    Q::unpack(gr[i], gv);
    const int64_t r = r0 + i;
    const bool inside = r >= ts.lo && r < ts.hi;
    const int32_t s = on ? ts.starts[sub * kRows + i] : -1;
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      float av, keep;
      gate_pair(gv[c], &av, &keep);
      float uv = keep * xv[c];
      if (s >= 0 && p.initial != nullptr) uv = fmaf(av, __ldg(p.initial + s * p.channels + col * kCh + c), uv);
      const bool restart = s >= 0 || !inside;
      a[i][c] = restart ? -1.0f : av;
      u[i][c] = inside ? uv : 0.0f;
      ph[c] = restart ? u[i][c] : fmaf(av, ph[c], uv);
      pa[c] = (restart || pa[c] < 0.0f) ? -1.0f : pa[c] * av;
    }
  }
  if (sub < p.geo.subs) {
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      sa[sub * chans + lc * kCh + c] = pa[c];
      sh[sub * chans + lc * kCh + c] = ph[c];
    }
  }
  __syncthreads();
  for (int ch = threadIdx.x; ch < chans; ch += kThreads) {
    float ta, th;
    compose(sa, sh, chans, p.geo.subs, false, ch, &ta, &th);
    const int64_t gc = static_cast<int64_t>(part) * chans + ch;
    if (PHASE == kAggregate && gc < p.channels) {
      p.agg_a[tile * p.channels + gc] = ta;
      p.agg_h[tile * p.channels + gc] = th;
    }
  }
  if (PHASE == kAggregate) return;
  __syncthreads();
  if (!on) return;
  float st[kCh];
#pragma unroll
  for (int c = 0; c < kCh; ++c) {
    st[c] = enter(sa[sub * chans + lc * kCh + c], sh[sub * chans + lc * kCh + c],
                  p.states[tile * p.channels + col * kCh + c]);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (r0 + i >= p.rows) break;
#pragma unroll
    for (int c = 0; c < kCh; ++c) st[c] = enter(a[i][c], u[i][c], st[c]);
    if (p.h != nullptr) static_cast<typename Q::raw*>(p.h)[(r0 + i) * p.geo.cols + col] = Q::pack(st);
    const int32_t s = ts.ends[sub * kRows + i];
    if (s >= 0 && p.final != nullptr) {
#pragma unroll
      for (int c = 0; c < kCh; ++c) p.final[s * p.channels + col * kCh + c] = st[c];
    }
  }
}

template <class T, int PHASE>
__global__ void __launch_bounds__(kThreads, 2) scan_backward_kernel(Params p) {
  using Q = Quad<T>;
  __shared__ TileSegments ts;
  __shared__ float sa[kThreads * kCh], sh[kThreads * kCh];
  const int32_t tile = static_cast<int32_t>(blockIdx.x / p.geo.across), part = blockIdx.x % p.geo.across;
  const int sub = threadIdx.x / p.geo.width, lc = threadIdx.x - sub * p.geo.width;
  const int col = part * p.geo.width + lc;
  const bool on = sub < p.geo.subs && col < p.geo.cols;
  const int64_t row0 = static_cast<int64_t>(tile) * p.geo.tile_rows;
  const int64_t r0 = row0 + static_cast<int64_t>(sub) * kRows;
  const int chans = p.geo.width * kCh;
  const int slot = sub * chans + lc * kCh;
  const typename Q::raw* x = static_cast<const typename Q::raw*>(p.x);
  const typename Q::raw* gate = static_cast<const typename Q::raw*>(p.gate);
  const typename Q::raw* grad = static_cast<const typename Q::raw*>(p.grad);

  typename Q::raw xr[kRows], gr[kRows], dr[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const bool ok = on && r0 + i < p.rows;
    gr[i] = ok ? __ldg(gate + (r0 + i) * p.geo.cols + col) : Q::zero();
    if (PHASE == kApply) xr[i] = ok ? __ldg(x + (r0 + i) * p.geo.cols + col) : Q::zero();
    dr[i] = ok && grad != nullptr ? __ldg(grad + (r0 + i) * p.geo.cols + col) : Q::zero();
  }
  find_segments(p, row0, p.geo.tile_rows, ts);

  float q[kRows][kCh];  // (h_{t-1} - x_t) a_t (1 - a_t)
  if (PHASE == kApply) {
    // The forward states again, from the state saved at the tile's edge.
    float pa[kCh], ph[kCh];
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      pa[c] = 1.0f;
      ph[c] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      float xv[kCh], gv[kCh];
      Q::unpack(xr[i], xv);
      Q::unpack(gr[i], gv);
      const int32_t s = on ? ts.starts[sub * kRows + i] : -1;
      const bool inside = r0 + i >= ts.lo && r0 + i < ts.hi;
      const bool restart = s >= 0 || !inside;
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        float av, keep;
        gate_pair(gv[c], &av, &keep);
        float uv = keep * xv[c];
        if (s >= 0 && p.initial != nullptr) uv = fmaf(av, __ldg(p.initial + s * p.channels + col * kCh + c), uv);
        ph[c] = restart ? (inside ? uv : 0.0f) : fmaf(av, ph[c], uv);
        pa[c] = (restart || pa[c] < 0.0f) ? -1.0f : pa[c] * av;
      }
    }
    if (sub < p.geo.subs) {
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        sa[slot + c] = pa[c];
        sh[slot + c] = ph[c];
      }
    }
    __syncthreads();
    for (int ch = threadIdx.x; ch < chans; ch += kThreads) {
      float ta, th;
      compose(sa, sh, chans, p.geo.subs, false, ch, &ta, &th);
    }
    __syncthreads();
    float st[kCh];
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      st[c] = on ? enter(sa[slot + c], sh[slot + c], p.saved[tile * p.channels + col * kCh + c]) : 0.0f;
    }
    __syncthreads();  // sa and sh are used again below
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      float xv[kCh], gv[kCh];
      Q::unpack(xr[i], xv);
      Q::unpack(gr[i], gv);
      const int32_t s = on ? ts.starts[sub * kRows + i] : -1;
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        float av, keep;
        gate_pair(gv[c], &av, &keep);
        if (s >= 0) st[c] = p.initial != nullptr ? __ldg(p.initial + s * p.channels + col * kCh + c) : 0.0f;
        q[i][c] = (st[c] - xv[c]) * (av * keep);
        st[c] = fmaf(av, st[c], keep * xv[c]);
      }
    }
  }

  // e_t = a_t (d_t + e_{t+1}) from the last row of the thread to its first.
  float a[kRows][kCh], d[kRows][kCh];
  float pa[kCh], pe[kCh];
#pragma unroll
  for (int c = 0; c < kCh; ++c) {
    pa[c] = 1.0f;
    pe[c] = 0.0f;
  }
#pragma unroll
  for (int i = kRows - 1; i >= 0; --i) {
    float gv[kCh], dv[kCh];
    Q::unpack(gr[i], gv);
    Q::unpack(dr[i], dv);
    const int32_t s = on ? ts.ends[sub * kRows + i] : -1;
    const bool inside = r0 + i >= ts.lo && r0 + i < ts.hi;
    const bool restart = s >= 0 || !inside;
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      float av, keep;
      gate_pair(gv[c], &av, &keep);
      if (s >= 0 && p.grad_final != nullptr) dv[c] += __ldg(p.grad_final + s * p.channels + col * kCh + c);
      a[i][c] = av;
      d[i][c] = inside ? dv[c] : 0.0f;
      pe[c] = inside ? av * (restart ? dv[c] : dv[c] + pe[c]) : 0.0f;
      pa[c] = (restart || pa[c] < 0.0f) ? -1.0f : pa[c] * av;
    }
  }
  if (sub < p.geo.subs) {
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      sa[slot + c] = pa[c];
      sh[slot + c] = pe[c];
    }
  }
  __syncthreads();
  for (int ch = threadIdx.x; ch < chans; ch += kThreads) {
    float ta, th;
    compose(sa, sh, chans, p.geo.subs, true, ch, &ta, &th);
    const int64_t gc = static_cast<int64_t>(part) * chans + ch;
    if (PHASE == kAggregate && gc < p.channels) {
      p.agg_a[tile * p.channels + gc] = ta;
      p.agg_h[tile * p.channels + gc] = th;
    }
  }
  if (PHASE == kAggregate) return;
  __syncthreads();
  if (!on) return;
  float e[kCh];
#pragma unroll
  for (int c = 0; c < kCh; ++c) {
    e[c] = enter(sa[slot + c], sh[slot + c], p.states[tile * p.channels + col * kCh + c]);
  }
#pragma unroll
  for (int i = kRows - 1; i >= 0; --i) {
    if (r0 + i >= p.rows) continue;
    const bool inside = r0 + i >= ts.lo && r0 + i < ts.hi;
    const bool last = ts.ends[sub * kRows + i] >= 0;
    float gv[kCh], dx[kCh], dg[kCh];
    Q::unpack(gr[i], gv);
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      float av, keep;
      gate_pair(gv[c], &av, &keep);
      const float delta = last ? d[i][c] : d[i][c] + e[c];
      e[c] = inside ? a[i][c] * delta : 0.0f;
      dx[c] = inside ? keep * delta : 0.0f;
      dg[c] = inside ? delta * q[i][c] : 0.0f;
    }
    static_cast<typename Q::raw*>(p.dx)[(r0 + i) * p.geo.cols + col] = Q::pack(dx);
    static_cast<typename Q::raw*>(p.dgate)[(r0 + i) * p.geo.cols + col] = Q::pack(dg);
    const int32_t s = ts.starts[sub * kRows + i];
    if (s >= 0 && p.dinitial != nullptr) {
#pragma unroll
      for (int c = 0; c < kCh; ++c) p.dinitial[s * p.channels + col * kCh + c] = e[c];
    }
  }
}

// States entering the tiles from their (A, H), one thread per channel.
__global__ void scan_states_kernel(Params p, int up) {
  const int64_t ch = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (ch >= p.channels) return;
  float st = 0.0f;
  for (int64_t k = 0; k < p.geo.tiles; ++k) {
    const int64_t i = (up ? p.geo.tiles - 1 - k : k) * p.channels + ch;
    p.states[i] = st;
    st = enter(p.agg_a[i], p.agg_h[i], st);
  }
}

// out[s] = in[s] (0 without `in`) for the segments without rows.
__global__ void empty_segments_kernel(const int64_t* __restrict__ off, int64_t nseg, int64_t channels,
                                      const float* __restrict__ in, float* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t s = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; s < nseg; s += warps) {
    if (off[s] < off[s + 1]) continue;
    for (int64_t c = lane; c < channels; c += 32) out[s * channels + c] = in != nullptr ? in[s * channels + c] : 0.0f;
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
  if (channels > (int64_t(1) << 20) || nseg >= (int64_t(1) << 31) ||
      geometry(rows, channels).tiles * geometry(rows, channels).across >= (int64_t(1) << 31)) {
    return fail(DGFX_ERR_UNSUPPORTED, std::string(who) + ": sizes out of range");
  }
  return DGFX_OK;
}

bool quad_aligned(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == DGFX_F32 ? 15u : 7u)) == 0;
}

unsigned warps_grid(int64_t warps) {
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(ceil_div(warps, 8), 148 * 8)));
}

struct Work {
  float *a, *h, *states;
  bool ok;
  size_t bytes;
};

Work carve(void* base, size_t cap, const Geometry& g, int64_t channels) {
  Arena arena(base, cap);
  const size_t n = static_cast<size_t>(g.tiles) * channels;
  Work w;
  w.a = arena.take<float>(n);
  w.h = arena.take<float>(n);
  w.states = arena.take<float>(n);
  w.ok = arena.ok();
  w.bytes = arena.used;
  return w;
}

}  // namespace
}  // namespace dgfx

using namespace dgfx;

extern "C" int dgfx_gated_scan_workspace_size(int64_t rows, int64_t channels, size_t* workspace_bytes,
                                              size_t* saved_bytes) {
  DGFX_TRY(check_shape("dgfx_gated_scan_workspace_size", rows, channels, 0, DGFX_F32));
  const Geometry g = geometry(rows, channels);
  if (workspace_bytes != nullptr) *workspace_bytes = carve(nullptr, 0, g, channels).bytes;
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
  if (!quad_aligned(d_x, dtype) || !quad_aligned(d_gate, dtype) || !quad_aligned(d_h, dtype)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_scan: operands must be aligned to 4 elements");
  }
  Params p{};
  p.geo = geometry(rows, channels);
  const Work w = carve(d_workspace, workspace_bytes, p.geo, channels);
  if (d_workspace == nullptr || !w.ok) return fail(DGFX_ERR_WORKSPACE, "dgfx_gated_scan: workspace too small");
  p.x = d_x;
  p.gate = d_gate;
  p.off = d_offsets;
  p.initial = d_initial;
  p.h = d_h;
  p.final = d_final;
  p.agg_a = w.a;
  p.agg_h = w.h;
  p.states = d_saved != nullptr ? d_saved : w.states;
  p.rows = rows;
  p.channels = channels;
  p.nseg = nseg;
  if (d_final != nullptr && nseg > 0) {
    empty_segments_kernel<<<warps_grid(nseg), 256, 0, stream>>>(d_offsets, nseg, channels, d_initial, d_final);
    DGFX_CUDA_TRY(cudaGetLastError());
  }
  if (rows == 0) return DGFX_OK;
  const unsigned grid = static_cast<unsigned>(p.geo.tiles * p.geo.across);
  const unsigned cgrid = static_cast<unsigned>(ceil_div(channels, 64));
  if (dtype == DGFX_F32) {
    scan_forward_kernel<float, kAggregate><<<grid, kThreads, 0, stream>>>(p);
    scan_states_kernel<<<cgrid, 64, 0, stream>>>(p, 0);
    scan_forward_kernel<float, kApply><<<grid, kThreads, 0, stream>>>(p);
  } else {
    scan_forward_kernel<__nv_bfloat16, kAggregate><<<grid, kThreads, 0, stream>>>(p);
    scan_states_kernel<<<cgrid, 64, 0, stream>>>(p, 0);
    scan_forward_kernel<__nv_bfloat16, kApply><<<grid, kThreads, 0, stream>>>(p);
  }
  DGFX_CUDA_TRY(cudaGetLastError());
  return DGFX_OK;
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
      !quad_aligned(d_dx, dtype) || !quad_aligned(d_dgate, dtype)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_scan_backward: operands must be aligned to 4 elements");
  }
  Params p{};
  p.geo = geometry(rows, channels);
  const Work w = carve(d_workspace, workspace_bytes, p.geo, channels);
  if (d_workspace == nullptr || !w.ok) return fail(DGFX_ERR_WORKSPACE, "dgfx_gated_scan_backward: workspace too small");
  p.x = d_x;
  p.gate = d_gate;
  p.off = d_offsets;
  p.initial = d_initial;
  p.grad = d_grad_h;
  p.grad_final = d_grad_final;
  p.dx = d_dx;
  p.dgate = d_dgate;
  p.dinitial = d_dinitial;
  p.agg_a = w.a;
  p.agg_h = w.h;
  p.states = w.states;
  p.saved = d_saved;
  p.rows = rows;
  p.channels = channels;
  p.nseg = nseg;
  if (d_dinitial != nullptr && nseg > 0) {
    empty_segments_kernel<<<warps_grid(nseg), 256, 0, stream>>>(d_offsets, nseg, channels, d_grad_final, d_dinitial);
    DGFX_CUDA_TRY(cudaGetLastError());
  }
  if (rows == 0) return DGFX_OK;
  const unsigned grid = static_cast<unsigned>(p.geo.tiles * p.geo.across);
  const unsigned cgrid = static_cast<unsigned>(ceil_div(channels, 64));
  if (dtype == DGFX_F32) {
    scan_backward_kernel<float, kAggregate><<<grid, kThreads, 0, stream>>>(p);
    scan_states_kernel<<<cgrid, 64, 0, stream>>>(p, 1);
    scan_backward_kernel<float, kApply><<<grid, kThreads, 0, stream>>>(p);
  } else {
    scan_backward_kernel<__nv_bfloat16, kAggregate><<<grid, kThreads, 0, stream>>>(p);
    scan_states_kernel<<<cgrid, 64, 0, stream>>>(p, 1);
    scan_backward_kernel<__nv_bfloat16, kApply><<<grid, kThreads, 0, stream>>>(p);
  }
  DGFX_CUDA_TRY(cudaGetLastError());
  return DGFX_OK;
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
