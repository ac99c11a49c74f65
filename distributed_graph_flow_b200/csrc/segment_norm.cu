// Group norm with an activation over the ragged segments of a merged batch,
// channels last (sm_100a).
//
// Segment s holds rows off[s] .. off[s+1] of x [rows, C]; group g holds C / G
// adjacent channels. Over the n = (rows of s) x (C / G) values of (s, g):
//   mean = sum x / n,  rstd = 1 / sqrt(sum (x - mean)^2 / n + eps),
//   z = (x - mean) rstd w_c + b_c,  y = act(z).
// Backward, with dz = dy act'(z), xhat = (x - mean) rstd:
//   dx = rstd (w dz - S1 / n - xhat S2 / n),  S1 = sum w dz,
//   S2 = sum w dz xhat (over (s, g)),  dw_c = sum dz xhat,  db_c = sum dz.
//
// Bound by HBM. A short segment (a sampled graph) is the work of a team of
// threads: it reads the segment for the sums and again for the result, the second
// time from L1 as long as the segments of an SM's teams fit there (the average one does; the
// largest that a team takes comes from L2). A team is the smallest power of two of threads (32 .. 512,
// at least a row) that reads the average segment in a few steps, so many
// small segments share a block. Segments of more than three to eight steps are
// listed and go through three more kernels: the first reads row
// tiles and leaves a mean and a centred sum of squares per tile and group, the
// second joins a segment's tiles, the third applies them, tiles in reverse
// order, so that what the first read last is still in L2.
// When no segment can be that long only the first kernel is launched.
//
// Thread t of a team takes the quad (4 channels) t mod Q of every (team / Q)-th
// row, Q = C / 4: loads are whole rows and a thread's channels never change,
// so weights and the sums for dw and db stay in registers. Squares are summed
// around a value of the segment, then around the means, never as sum x^2 -
// mean^2. All sums are fp32 in an order fixed by the sizes: results do not change from run to
// run. Rows outside [off[0], off[nseg]) are written as zeros and their inputs
// are never used.
//
// Measured (L2 flushed, forward + backward unless said): one segment of a
// million rows x 256 bf16 channels, 16 groups, silu 784 us: x is read twice on the
// way forward, x and dy twice on the way back, 4.1 GB in all, 5.2 TB/s; 300 ragged
// segments in 250,001 rows x 200 fp32, gelu 375 us (1.6 GB); a merged batch of
// 1024 graphs, 41,003 rows x 256 bf16, relu, forward 37 us: one segment per team,
// so the longest one's chain of loads and sums and the five launches are what it
// takes. Segments of a single row run far below HBM: a team's fixed work per segment
// decides (a million rows x 64 bf16, one group: forward 1.26 ms, 0.2 TB/s; x 256
// 2.26 ms, 0.45 TB/s). At its 80 registers norm_backward_kernel spills 56 to 100
// bytes per thread with an activation in bf16 (8 without), 40 to 64 in fp32 (but for none
// and relu); norm_forward_kernel spills 20 with gelu in bf16, the tile kernels up to 16.
#include <algorithm>
#include <string>

#include "layer_math.cuh"

namespace dgfx {
namespace {

constexpr int kSms = 148;
constexpr int kCh = 4;

// Rows loaded at a time: 128 bytes per thread in all.
template <class T>
constexpr int kAhead = sizeof(T) == 2 ? 16 : 8;

struct Params {
  const void* x;
  const void* dy;
  const int64_t* off;
  const float* weight;
  const float* bias;
  void* y;  // output, or dx going backward
  float* mean;
  float* rstd;
  float* partial;  // backward: [blocks, 2, C], dw and db of one block
  // Long segments (null if none can be long): how many and how many tiles
  // (count << 32 | tiles), the list (rows, number, first tile), per tile and
  // group two sums.
  unsigned long long* long_counter;
  longlong2* long_span;  // first row, rows
  int32_t* long_seg;
  int32_t* long_base;
  float2* tile_sums;
  float2* seg_sums;  // backward: S1 / n and S2 / n per long segment and group
  int64_t rows, nseg;
  int64_t loop_rows;  // rows of the longest segment that one team takes
  int64_t tile_rows;
  int64_t max_long, max_tiles;  // room of the list and of tile_sums
  int32_t channels, groups, quads;
  int32_t team;       // threads per team of the short-segment kernels
  int32_t split;      // values a thread gives to the group sums: 1 if a quad lies in one group, else 4
  int32_t blocks_before;  // backward: partial slots of the short-segment kernel
  float eps;
};

// A thread's four channels as two pairs.
struct Pairs {
  float2 v[2];
  __device__ Pairs() {}
  __device__ explicit Pairs(const float (&f)[kCh]) {
    v[0] = make_float2(f[0], f[1]);
    v[1] = make_float2(f[2], f[3]);
  }
  __device__ void to(float (&f)[kCh]) const {
    f[0] = v[0].x;
    f[1] = v[0].y;
    f[2] = v[1].x;
    f[3] = v[1].y;
  }
};

__device__ __forceinline__ Pairs negated(const float (&f)[kCh]) {
  const float n[kCh] = {-f[0], -f[1], -f[2], -f[3]};
  return Pairs(n);
}

template <class T>
__device__ __forceinline__ Pairs unpack_pairs(const typename Quad<T>::raw& r) {
  float f[kCh];
  Quad<T>::unpack(r, f);
  return Pairs(f);
}

struct Place {
  int rl, col, per_pass;
  bool on;
  __device__ Place(const Params& p, int t, int threads) {
    per_pass = threads / p.quads;
    rl = t / p.quads;
    col = t - rl * p.quads;
    on = rl < per_pass;
  }
};

__device__ __forceinline__ void team_sync(int id, int threads) {
  if (threads == 32) {
    __syncwarp();
    return;
  }
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Sums of acc[k][c] over the team's rows and each group's channels into
// gsum[k * groups + g], there for the whole team after the call. red holds
// K * team * split floats; a group's values are contiguous in it, and
// 1 .. 32 neighbouring lanes add them up.
template <int K>
__device__ __forceinline__ void group_sums(const Params& p, const float (&acc)[K][kCh], const Place& at, int t,
                                           int threads, int bar, float* red, float* gsum) {
  const int values = p.quads * p.split * at.per_pass;  // of one k
  if (at.on) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (p.split == 1) {
        red[k * values + at.col * at.per_pass + at.rl] = (acc[k][0] + acc[k][1]) + (acc[k][2] + acc[k][3]);
      } else {
#pragma unroll
        for (int c = 0; c < kCh; ++c) red[k * values + (at.col * kCh + c) * at.per_pass + at.rl] = acc[k][c];
      }
    }
  }
  team_sync(bar, threads);
  // Lanes per group: a power of two of at most 32.
  const int spare = threads / (K * p.groups);
  const int shift = spare >= 32 ? 5 : (spare < 1 ? 0 : 31 - __clz(spare));
  const int lanes = 1 << shift;
  const int each = values / p.groups;
  const int sub = t & (lanes - 1);
  for (int i = 0; i < (K * p.groups) << shift; i += threads) {
    const int g = (t + i) >> shift;  // k * groups + group
    float s = 0.0f;
    if (g < K * p.groups) {
      for (int e = sub; e < each; e += lanes) s += red[g * each + e];
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (g < K * p.groups && sub == 0) gsum[g] = s;
  }
  team_sync(bar, threads);
}

// The affine parameters of this thread's channels.
struct Affine {
  float w[kCh], b[kCh];
  __device__ Affine(const Params& p, const Place& at) {
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      const int ch = at.on ? at.col * kCh + c : 0;
      w[c] = p.weight != nullptr ? __ldg(p.weight + ch) : 1.0f;
      b[c] = p.bias != nullptr ? __ldg(p.bias + ch) : 0.0f;
    }
  }
};

// Calls f(c, group of channel c) for this thread's channels. g0 is the group
// of the first; only a quad that crosses groups divides again.
template <class F>
__device__ __forceinline__ void each_group(const Params& p, const Place& at, int g0, F f) {
  if (p.split == 1) {
#pragma unroll
    for (int c = 0; c < kCh; ++c) f(c, g0);
  } else {
    const int cg = p.channels / p.groups;
#pragma unroll
    for (int c = 0; c < kCh; ++c) f(c, (at.col * kCh + c) / cg);
  }
}

// Zeros in the rows outside of every segment: written by the last kernel of a
// call, whose grid covers the GPU where there are many rows (by the first one,
// with a block per few segments, 6576 spare rows of 328 channels took 50 us).
template <class T>
__device__ __forceinline__ void zero_outside(const Params& p) {
  const int64_t lo = clamp64(p.off[0], 0, p.rows), hi = clamp64(p.off[p.nseg], lo, p.rows);
  auto* y = static_cast<typename Quad<T>::raw*>(p.y);
  const int64_t threads = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t i = t; i < lo * p.quads; i += threads) y[i] = Quad<T>::zero();
  for (int64_t i = hi * p.quads + t; i < p.rows * p.quads; i += threads) y[i] = Quad<T>::zero();
}

// The segments of more than loop_rows rows, each with its rows and its first
// tile, in an order that the offsets fix. One block: a thread counts in its
// share of the segments, then writes behind what the threads before it have. It runs beside the
// short-segment kernel, which needs nothing of it (a list made by that one's
// last block, from slots that had to be cleared before, took 42 instead of 37 us
// for a merged batch of 1024 graphs).
__global__ void __launch_bounds__(1024) norm_list_kernel(Params p) {
  let_next_start();
  __shared__ unsigned long long smem[33];
  const int64_t lo = clamp64(p.off[0], 0, p.rows), hi = clamp64(p.off[p.nseg], lo, p.rows);
  auto visit = [&](auto f) {
    constexpr int N = 8;  // segments at a time, blockDim apart: loads of neighbours
    for (int64_t s0 = threadIdx.x; s0 < p.nseg; s0 += N * blockDim.x) {
      int64_t begin[N], end[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t s = s0 + i * blockDim.x;
        begin[i] = end[i] = 0;
        if (s < p.nseg) {
          begin[i] = __ldg(p.off + s);
          end[i] = __ldg(p.off + s + 1);
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t b = clamp64(begin[i], lo, hi), n = clamp64(end[i], b, hi) - b;
        if (n > p.loop_rows) {
          f(s0 + i * blockDim.x, b, n, (1ull << 32) | static_cast<unsigned long long>((n + p.tile_rows - 1) / p.tile_rows));
        }
      }
    }
  };
  unsigned long long mine = 0, all = 0;  // count << 32 | tiles
  visit([&](int64_t, int64_t, int64_t, unsigned long long add) { mine += add; });
  unsigned long long at = block_exclusive_scan(mine, smem, &all);
  if (mine != 0) visit([&](int64_t s, int64_t b, int64_t n, unsigned long long add) {
    const int64_t i = static_cast<int64_t>(at >> 32), base = static_cast<int64_t>(at & 0xffffffffull);
    if (i < p.max_long) {  // ascending offsets fit; others stay inside of the tables
      p.long_span[i] = make_longlong2(b, n);
      p.long_seg[i] = static_cast<int32_t>(s);
      p.long_base[i] = static_cast<int32_t>(base < p.max_tiles ? base : p.max_tiles);
    }
    at += add;
  });
  if (threadIdx.x == 0) *p.long_counter = all;
}

struct LongList {
  int count, tiles;
  __device__ explicit LongList(const Params& p) {
    const unsigned long long c = *p.long_counter;
    const int64_t t = static_cast<int64_t>(c & 0xffffffffull);
    const int64_t n = static_cast<int64_t>(c >> 32);
    count = static_cast<int>(n < p.max_long ? n : p.max_long);
    tiles = static_cast<int>(t < p.max_tiles ? t : p.max_tiles);
  }
};

// The listed segment that holds `tile`: the last one whose first tile is not
// past it. Every lane of a warp probes one of 32 evenly spaced entries.
__device__ __forceinline__ int find_long(const int32_t* base, int count, int tile) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int q = lo + step * lane;
    const bool le = q < hi && base[q] <= tile;
    const int k = 31 - __clz(static_cast<int>(__ballot_sync(0xffffffffu, le)));
    hi = min(hi, lo + step * (k + 1));
    lo = lo + step * k;
  }
  return lo;
}

// This thread's share of rows [begin, end): `mine` rows of its lane from
// element `first` on, `pitch` elements (quads) apart.
struct Share {
  int64_t first;
  int mine, pitch;
  __device__ Share(const Params& p, const Place& at, int64_t begin, int64_t end) {
    first = (begin + at.rl) * p.quads + at.col;
    const int n = static_cast<int>(end - begin);
    mine = at.on && n > at.rl ? (n - at.rl + at.per_pass - 1) / at.per_pass : 0;
    pitch = at.per_pass * p.quads;
  }
};

// Calls f(quad of x) or f(quad of x, quad of d) for `left` <= N rows, all
// loads first.
template <class T, int N, class F>
__device__ __forceinline__ void few_rows(const typename Quad<T>::raw* x, int pitch, int left, F f) {
  typename Quad<T>::raw v[N];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = i < left ? __ldg(x + i * pitch) : Quad<T>::zero();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i < left) f(v[i]);
  }
}
template <class T, int N, class F>
__device__ __forceinline__ void few_rows(const typename Quad<T>::raw* x, const typename Quad<T>::raw* d, int pitch, int left,
                                         F f) {
  typename Quad<T>::raw v[N], w[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = i < left ? __ldg(x + i * pitch) : Quad<T>::zero();
    w[i] = i < left ? __ldg(d + i * pitch) : Quad<T>::zero();
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i < left) f(v[i], w[i]);
  }
}

// The same for a share's rows in order, kAhead loads at a time. WIDE: full
// batches without checks, then the rest; otherwise one checked batch of half as
// many, over and over: a short segment has few full batches, and its warps,
// each somewhere else in the code, live off the instruction cache.
template <class T, bool WIDE, class F>
__device__ __forceinline__ void each_row(const Share& sh, const void* base, F f) {
  constexpr int B = WIDE ? kAhead<T> : kAhead<T> / 2;
  using raw = typename Quad<T>::raw;
  const raw* x = static_cast<const raw*>(base) + sh.first;
  int left = sh.mine;
  if (WIDE) {
    for (; left >= B; left -= B) {
      raw v[B];
#pragma unroll
      for (int i = 0; i < B; ++i) v[i] = __ldg(x + i * sh.pitch);
      x += B * sh.pitch;
#pragma unroll
      for (int i = 0; i < B; ++i) f(v[i]);
    }
    if (left > B / 4) few_rows<T, B - 1>(x, sh.pitch, left, f);
    else if (left > 0) few_rows<T, B / 4>(x, sh.pitch, left, f);
  } else {
#pragma unroll 1
    for (; left > 0; left -= B) {
      few_rows<T, B>(x, sh.pitch, left, f);
      x += B * sh.pitch;
    }
  }
}
template <class T, bool WIDE, class F>
__device__ __forceinline__ void each_row(const Share& sh, const void* base, const void* other, F f) {
  constexpr int B = kAhead<T> / 2;
  using raw = typename Quad<T>::raw;
  const raw* x = static_cast<const raw*>(base) + sh.first;
  const raw* d = static_cast<const raw*>(other) + sh.first;
  int left = sh.mine;
  if (WIDE) {
    for (; left >= B; left -= B) {
      raw v[B], w[B];
#pragma unroll
      for (int i = 0; i < B; ++i) {
        v[i] = __ldg(x + i * sh.pitch);
        w[i] = __ldg(d + i * sh.pitch);
      }
      x += B * sh.pitch;
      d += B * sh.pitch;
#pragma unroll
      for (int i = 0; i < B; ++i) f(v[i], w[i]);
    }
    if (left > B / 4) few_rows<T, B - 1>(x, d, sh.pitch, left, f);
    else if (left > 0) few_rows<T, B / 4>(x, d, sh.pitch, left, f);
  } else {
#pragma unroll 1
    for (; left > 0; left -= B) {
      few_rows<T, B>(x, d, sh.pitch, left, f);
      x += B * sh.pitch;
      d += B * sh.pitch;
    }
  }
}

// Mean and centred squares of this thread's channels over its share. The
// sums run around the share's first row x0: with d = x - x0, the centred squares
// are sum d^2 - (sum d)^2 / n. What that loses is at most about n 2^-24 of
// sum d^2, and as x0 is one of the values, n (x0 - mean)^2 summed over the
// threads is at most n times the segment's own centred squares: a relative error of n 2^-24,
// n the rows of a thread, however far the mean is from zero.
struct RowStats {
  float mean[kCh], m2[kCh], have;
};

template <class T, bool WIDE>
__device__ __forceinline__ RowStats row_stats(const Params& p, const Share& sh) {
  using Q = Quad<T>;
  RowStats s = {};
  if (sh.mine == 0) return s;
  float x0[kCh];
  Pairs minus;
  Pairs sum(s.mean), sq(s.m2);
  bool first = true;
  each_row<T, WIDE>(sh, p.x, [&](const typename Q::raw& v) {
    const Pairs f = unpack_pairs<T>(v);
    if (first) {
      f.to(x0);
      minus = negated(x0);
      first = false;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float2 d = add2(f.v[c], minus.v[c]);
      sum.v[c] = add2(sum.v[c], d);
      sq.v[c] = fma2(d, d, sq.v[c]);
    }
  });
  sum.to(s.mean);
  sq.to(s.m2);
  s.have = static_cast<float>(sh.mine);
  const float inv = 1.0f / s.have;
#pragma unroll
  for (int c = 0; c < kCh; ++c) {
    const float d = s.mean[c] * inv;
    const float m2 = s.m2[c] - s.mean[c] * d;
    s.m2[c] = m2 < 0.0f ? 0.0f : m2;
    s.mean[c] = x0[c] + d;
  }
  return s;
}

// y of a share's rows from their statistics.
template <class T, int ACT, bool WIDE>
__device__ __forceinline__ void apply_rows(const Params& p, const Share& sh, const Affine& af, const float (&mu)[kCh],
                                           const float (&rs)[kCh]) {
  using Q = Quad<T>;
  if (sh.mine == 0) return;
  float scale[kCh];
#pragma unroll
  for (int c = 0; c < kCh; ++c) scale[c] = rs[c] * af.w[c];
  const Pairs minus = negated(mu), sc(scale), shift(af.b);
  typename Q::raw* y = static_cast<typename Q::raw*>(p.y) + sh.first;
  each_row<T, WIDE>(sh, p.x, [&](const typename Q::raw& v) {
    Pairs f = unpack_pairs<T>(v);
#pragma unroll
    for (int c = 0; c < 2; ++c) f.v[c] = act2_f<ACT>(fma2(add2(f.v[c], minus.v[c]), sc.v[c], shift.v[c]));
    float o[kCh];
    f.to(o);
    *y = Q::pack(o);
    y += sh.pitch;
  });
}

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
template <class T, int ACT>
__global__ void __maxnreg__(64) norm_forward_kernel(Params p) {
  let_next_start();
  extern __shared__ float smem[];
  const int in_block = threadIdx.x / p.team, t = threadIdx.x - in_block * p.team, bar = 1 + in_block;
  const Place at(p, t, p.team);
  const int g0 = at.col * kCh / (p.channels / p.groups);
  float* red = smem + in_block * (p.team * p.split + p.groups);
  float* gsum = red + p.team * p.split;
  const int64_t lo = clamp64(p.off[0], 0, p.rows), hi = clamp64(p.off[p.nseg], lo, p.rows);
  const int cg = p.channels / p.groups;
  const Affine af(p, at);
  const int teams = blockDim.x / p.team;
  for (int64_t s = static_cast<int64_t>(blockIdx.x) * teams + in_block; s < p.nseg;
       s += static_cast<int64_t>(gridDim.x) * teams) {
    const int64_t begin = clamp64(p.off[s], lo, hi), end = clamp64(p.off[s + 1], begin, hi);
    if (end - begin > p.loop_rows) continue;
    const int n = static_cast<int>(end - begin);
    if (n == 0) {
      for (int g = t; g < p.groups; g += p.team) {
        p.mean[s * p.groups + g] = 0.0f;
        p.rstd[s * p.groups + g] = rsqrtf(p.eps);
      }
      continue;
    }
    const float count = static_cast<float>(n) * static_cast<float>(cg), inv = 1.0f / count;
    float mu[kCh], rs[kCh], acc[1][kCh] = {};
    const Share sh(p, at, begin, end);
    const RowStats rst = row_stats<T, false>(p, sh);
#pragma unroll
    for (int c = 0; c < kCh; ++c) acc[0][c] = rst.have * rst.mean[c];
    group_sums<1>(p, acc, at, t, p.team, bar, red, gsum);
    each_group(p, at, g0, [&](int c, int g) {
      // A division: small segments of near values multiply the mean's rounding.
      mu[c] = at.on ? gsum[g] / count : 0.0f;
      const float d = rst.have > 0.0f ? rst.mean[c] - mu[c] : 0.0f;
      acc[0][c] = rst.m2[c] + rst.have * d * d;
    });
    for (int g = t; g < p.groups; g += p.team) p.mean[s * p.groups + g] = gsum[g] / count;
    // Its first barrier also ends the reads of gsum above.
    group_sums<1>(p, acc, at, t, p.team, bar, red, gsum);
    each_group(p, at, g0, [&](int c, int g) { rs[c] = at.on ? rsqrtf(gsum[g] * inv + p.eps) : 0.0f; });
    for (int g = t; g < p.groups; g += p.team) p.rstd[s * p.groups + g] = rsqrtf(gsum[g] * inv + p.eps);
    apply_rows<T, ACT, false>(p, sh, af, mu, rs);
  }
  // Behind the list kernel, which need not have ended before: whatever follows
  // this kernel then follows both.
  if (p.long_counter != nullptr) after_previous();
  else zero_outside<T>(p);
}

// One row tile of a listed segment.
struct Tile {
  int entry;
  int64_t seg, begin, end;  // rows [begin, end)
  __device__ Tile(const Params& p, const LongList& all, int tile) {
    entry = find_long(p.long_base, all.count, tile);
    seg = p.long_seg[entry];
    const longlong2 span = p.long_span[entry];
    const int64_t e = span.x + span.y;
    begin = span.x + static_cast<int64_t>(tile - p.long_base[entry]) * p.tile_rows;
    end = begin + p.tile_rows < e ? begin + p.tile_rows : e;
  }
};

template <class T>
__global__ void __maxnreg__(64) norm_tile_stats_kernel(Params p) {
  let_next_start();
  after_previous();
  extern __shared__ float smem[];
  float* red = smem;
  float* gsum = red + blockDim.x * p.split;
  const int threads = blockDim.x;
  const Place at(p, threadIdx.x, threads);
  const int g0 = at.col * kCh / (p.channels / p.groups);
  const LongList all(p);
  const int cg = p.channels / p.groups;
  for (int tile = blockIdx.x; tile < all.tiles; tile += gridDim.x) {
    const Tile tl(p, all, tile);
    const RowStats rst = row_stats<T, true>(p, Share(p, at, tl.begin, tl.end));
    const float n_tile = static_cast<float>(tl.end - tl.begin) * static_cast<float>(cg);
    float acc[1][kCh];
#pragma unroll
    for (int c = 0; c < kCh; ++c) acc[0][c] = rst.have * rst.mean[c];
    group_sums<1>(p, acc, at, threadIdx.x, threads, 1, red, gsum);
    each_group(p, at, g0, [&](int c, int g) {
      const float d = rst.have > 0.0f ? rst.mean[c] - gsum[g] / n_tile : 0.0f;
      acc[0][c] = rst.m2[c] + rst.have * d * d;
    });
    for (int g = threadIdx.x; g < p.groups; g += threads) {
      p.tile_sums[static_cast<int64_t>(tile) * p.groups + g].x = gsum[g] / n_tile;
    }
    group_sums<1>(p, acc, at, threadIdx.x, threads, 1, red, gsum);
    for (int g = threadIdx.x; g < p.groups; g += threads) {
      p.tile_sums[static_cast<int64_t>(tile) * p.groups + g].y = gsum[g];
    }
  }
}

// Joins the tiles of every listed segment: up to 32 groups per block and step,
// the tiles dealt to up to 32 lanes of threads, whose sums are added in order.
// Forward: means and centred squares, around the first tile's mean as the
// threads did their rows. BACKWARD: S1 / n and S2 / n. (One block per segment,
// the one that finished its last tile, took 0.4 ms for 256 groups of a million rows.)
template <bool BACKWARD>
__global__ void __launch_bounds__(256) norm_merge_kernel(Params p) {
  let_next_start();
  after_previous();
  __shared__ float2 part[256];
  constexpr int N = 8;  // loads at a time
  const LongList all(p);
  const int width = min(p.groups, 32), lanes = min(256 / width, 32), blocks = (p.groups + width - 1) / width;
  const int lane = threadIdx.x / width, col = threadIdx.x - lane * width;
  const int64_t cg = p.channels / p.groups;
  for (int64_t item = blockIdx.x; item < static_cast<int64_t>(all.count) * blocks; item += gridDim.x) {
    const int entry = static_cast<int>(item / blocks);
    const int g = static_cast<int>(item - static_cast<int64_t>(entry) * blocks) * width + col;
    const int first = p.long_base[entry], tiles = (entry + 1 < all.count ? p.long_base[entry + 1] : all.tiles) - first;
    const int64_t rows = p.long_span[entry].y, seg = p.long_seg[entry];
    if (tiles <= 0) continue;  // only where offsets do not ascend
    const float2* sums = p.tile_sums + static_cast<int64_t>(first) * p.groups + g;
    const float n_full = static_cast<float>(p.tile_rows) * static_cast<float>(cg);
    const float n_last = static_cast<float>(rows - (tiles - 1) * p.tile_rows) * static_cast<float>(cg);
    const bool on = lane < lanes && g < p.groups;
    float2 total = make_float2(0.0f, 0.0f), s0 = total;
    if (on) {
      if (!BACKWARD) s0 = sums[0];
      for (int k0 = lane; k0 < tiles; k0 += N * lanes) {
        float2 v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (k0 + i * lanes < tiles) v[i] = sums[static_cast<int64_t>(k0 + i * lanes) * p.groups];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int k = k0 + i * lanes;
          if (k < tiles) {
            if (BACKWARD) {
              total = add2(total, v[i]);
            } else {
              const float d = v[i].x - s0.x, n = k == tiles - 1 ? n_last : n_full;
              total.x += n * d;
              total.y += v[i].y + n * d * d;
            }
          }
        }
      }
    }
    part[threadIdx.x] = total;
    __syncthreads();
    if (on && lane == 0) {
      for (int k = 1; k < lanes; ++k) total = add2(total, part[k * width + col]);
      const float n_all = static_cast<float>(rows) * static_cast<float>(cg);
      if (BACKWARD) {
        p.seg_sums[static_cast<int64_t>(entry) * p.groups + g] = make_float2(total.x / n_all, total.y / n_all);
      } else {
        const float d = total.x / n_all, m2 = total.y - total.x * d;
        p.mean[seg * p.groups + g] = s0.x + d;
        p.rstd[seg * p.groups + g] = rsqrtf((m2 < 0.0f ? 0.0f : m2) / n_all + p.eps);
      }
    }
    __syncthreads();
  }
}

template <class T, int ACT>
__global__ void __maxnreg__(64) norm_tile_apply_kernel(Params p) {
  after_previous();
  zero_outside<T>(p);
  const Place at(p, threadIdx.x, blockDim.x);
  const int g0 = at.col * kCh / (p.channels / p.groups);
  const Affine af(p, at);
  const LongList all(p);
  for (int tile = all.tiles - 1 - static_cast<int>(blockIdx.x); tile >= 0; tile -= gridDim.x) {
    const Tile tl(p, all, tile);
    if (!at.on) continue;
    float mu[kCh], rs[kCh];
    each_group(p, at, g0, [&](int c, int g) {
      mu[c] = p.mean[tl.seg * p.groups + g];
      rs[c] = p.rstd[tl.seg * p.groups + g];
    });
    apply_rows<T, ACT, true>(p, Share(p, at, tl.begin, tl.end), af, mu, rs);
  }
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------
// xhat and dz of a pair. dz and w dz are rounded before any sum or
// subtraction, the same values in the sums and in dx: a segment of one value
// then cancels to zero exactly.
template <int ACT>
__device__ __forceinline__ void grad_terms(float2 x, float2 dy, float2 minus_mu, float2 rs, float2 w, float2 b,
                                           float2* xhat, float2* dz) {
  *xhat = mul2(add2(x, minus_mu), rs);
  float2 v, slope;
  act2_both_f<ACT>(fma2(*xhat, w, b), &v, &slope);
  *dz = mul2(dy, slope);
}

// This block's sums for dw and db over its threads, in order, to its slot.
__device__ __forceinline__ void write_partial(const Params& p, const float (&dwb)[2][kCh], const Place& at, int teams,
                                              int in_block, float* red, int slot) {
  __syncthreads();
  const int lanes = teams * at.per_pass;  // threads that share a column
  if (at.on) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        red[(k * lanes + in_block * at.per_pass + at.rl) * p.channels + at.col * kCh + c] = dwb[k][c];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.channels; i += blockDim.x) {
    const int k = i / p.channels, c = i - k * p.channels;
    float s = 0.0f;
    for (int r = 0; r < lanes; ++r) s += red[(k * lanes + r) * p.channels + c];
    p.partial[(static_cast<int64_t>(slot) * 2 + k) * p.channels + c] = s;
  }
}

// A share's sums for dw and db (added to dwb), and from them its part of the
// group sums: sum w dz xhat and sum w dz are w times those, channel by channel.
template <class T, int ACT, bool WIDE>
__device__ __forceinline__ void grad_sums(const Params& p, const Share& sh, const float (&mu)[kCh], const float (&rs)[kCh],
                                          const Affine& af, float (&acc)[2][kCh], float (&dwb)[2][kCh]) {
  using Q = Quad<T>;
  float dw[kCh] = {}, db[kCh] = {};  // these rows', so that long sums stay pairwise
  Pairs sw(dw), sb(db);
  const Pairs minus = negated(mu), r(rs), w(af.w), b(af.b);
  each_row<T, WIDE>(sh, p.x, p.dy, [&](const typename Q::raw& v, const typename Q::raw& d) {
    const Pairs f = unpack_pairs<T>(v), g = unpack_pairs<T>(d);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float2 xh, dz;
      grad_terms<ACT>(f.v[c], g.v[c], minus.v[c], r.v[c], w.v[c], b.v[c], &xh, &dz);
      sw.v[c] = fma2(dz, xh, sw.v[c]);
      sb.v[c] = add2(sb.v[c], dz);
    }
  });
  sw.to(dw);
  sb.to(db);
#pragma unroll
  for (int c = 0; c < kCh; ++c) {
    dwb[0][c] += dw[c];
    dwb[1][c] += db[c];
    acc[0][c] = __fmul_rn(db[c], af.w[c]);
    acc[1][c] = __fmul_rn(dw[c], af.w[c]);
  }
}

// dx of a share's rows from their group's sums (divided by n).
template <class T, int ACT, bool WIDE>
__device__ __forceinline__ void grad_rows(const Params& p, const Share& sh, const float (&mu)[kCh], const float (&rs)[kCh],
                                          const Affine& af, const float (&s1)[kCh], const float (&s2)[kCh]) {
  using Q = Quad<T>;
  typename Q::raw* dx = static_cast<typename Q::raw*>(p.y) + sh.first;
  const Pairs minus = negated(mu), r(rs), w(af.w), b(af.b), m1 = negated(s1), m2 = negated(s2);
  each_row<T, WIDE>(sh, p.x, p.dy, [&](const typename Q::raw& v, const typename Q::raw& d) {
    Pairs f = unpack_pairs<T>(v);
    const Pairs g = unpack_pairs<T>(d);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float2 xh, dz;
      grad_terms<ACT>(f.v[c], g.v[c], minus.v[c], r.v[c], w.v[c], b.v[c], &xh, &dz);
      // Scalar products: a packed one would be fused with the addition behind it.
      const float2 wdz = make_float2(__fmul_rn(dz.x, w.v[c].x), __fmul_rn(dz.y, w.v[c].y));
      f.v[c] = mul2(r.v[c], fma2(xh, m2.v[c], add2(wdz, m1.v[c])));
    }
    float o[kCh];
    f.to(o);
    *dx = Q::pack(o);
    dx += sh.pitch;
  });
}

template <class T, int ACT>
__global__ void __maxnreg__(80) norm_backward_kernel(Params p) {
  let_next_start();
  extern __shared__ float smem[];
  const int in_block = threadIdx.x / p.team, t = threadIdx.x - in_block * p.team, bar = 1 + in_block;
  const Place at(p, t, p.team);
  const int g0 = at.col * kCh / (p.channels / p.groups);
  float* red = smem + in_block * 2 * (p.team * p.split + p.groups);
  float* gsum = red + 2 * p.team * p.split;
  const int64_t lo = clamp64(p.off[0], 0, p.rows), hi = clamp64(p.off[p.nseg], lo, p.rows);
  const Affine af(p, at);
  const int cg = p.channels / p.groups;
  const int teams = blockDim.x / p.team;
  float dwb[2][kCh] = {};
  for (int64_t s = static_cast<int64_t>(blockIdx.x) * teams + in_block; s < p.nseg;
       s += static_cast<int64_t>(gridDim.x) * teams) {
    const int64_t begin = clamp64(p.off[s], lo, hi), end = clamp64(p.off[s + 1], begin, hi);
    if (begin == end) continue;
    if (end - begin > p.loop_rows) continue;
    const int n = static_cast<int>(end - begin);
    const float inv = 1.0f / (static_cast<float>(n) * static_cast<float>(cg));
    float mu[kCh], rs[kCh], acc[2][kCh] = {};
    each_group(p, at, g0, [&](int c, int g) {
      mu[c] = at.on ? __ldg(p.mean + s * p.groups + g) : 0.0f;
      rs[c] = at.on ? __ldg(p.rstd + s * p.groups + g) : 0.0f;
    });
    const Share sh(p, at, begin, end);
    grad_sums<T, ACT, false>(p, sh, mu, rs, af, acc, dwb);
    group_sums<2>(p, acc, at, t, p.team, bar, red, gsum);
    if (sh.mine > 0) {
      float s1[kCh], s2[kCh];
      each_group(p, at, g0, [&](int c, int g) {
        s1[c] = gsum[g] * inv;
        s2[c] = gsum[p.groups + g] * inv;
      });
      grad_rows<T, ACT, false>(p, sh, mu, rs, af, s1, s2);
    }
  }
  write_partial(p, dwb, at, teams, in_block, smem, blockIdx.x);
  if (p.long_counter != nullptr) after_previous();  // as in the forward kernel
  else zero_outside<T>(p);
}

template <class T, int ACT>
__global__ void __maxnreg__(80) norm_tile_grad_kernel(Params p) {
  let_next_start();
  after_previous();
  extern __shared__ float smem[];
  float* red = smem;
  float* gsum = red + 2 * blockDim.x * p.split;
  const int threads = blockDim.x;
  const Place at(p, threadIdx.x, threads);
  const int g0 = at.col * kCh / (p.channels / p.groups);
  const Affine af(p, at);
  const LongList all(p);
  const int cg = p.channels / p.groups;
  float dwb[2][kCh] = {};
  for (int tile = blockIdx.x; tile < all.tiles; tile += gridDim.x) {
    const Tile tl(p, all, tile);
    float mu[kCh], rs[kCh], acc[2][kCh] = {};
    each_group(p, at, g0, [&](int c, int g) {
      mu[c] = at.on ? __ldg(p.mean + tl.seg * p.groups + g) : 0.0f;
      rs[c] = at.on ? __ldg(p.rstd + tl.seg * p.groups + g) : 0.0f;
    });
    grad_sums<T, ACT, true>(p, Share(p, at, tl.begin, tl.end), mu, rs, af, acc, dwb);
    group_sums<2>(p, acc, at, threadIdx.x, threads, 1, red, gsum);
    for (int g = threadIdx.x; g < p.groups; g += threads) {
      p.tile_sums[static_cast<int64_t>(tile) * p.groups + g] = make_float2(gsum[g], gsum[p.groups + g]);
    }
  }
  write_partial(p, dwb, at, 1, 0, smem, p.blocks_before + blockIdx.x);
}

template <class T, int ACT>
__global__ void __maxnreg__(80) norm_tile_grad_apply_kernel(Params p) {
  let_next_start();
  after_previous();
  zero_outside<T>(p);
  const Place at(p, threadIdx.x, blockDim.x);
  const int g0 = at.col * kCh / (p.channels / p.groups);
  const Affine af(p, at);
  const LongList all(p);
  for (int tile = all.tiles - 1 - static_cast<int>(blockIdx.x); tile >= 0; tile -= gridDim.x) {
    const Tile tl(p, all, tile);
    if (!at.on) continue;
    float mu[kCh], rs[kCh], s1[kCh], s2[kCh];
    each_group(p, at, g0, [&](int c, int g) {
      mu[c] = __ldg(p.mean + tl.seg * p.groups + g);
      rs[c] = __ldg(p.rstd + tl.seg * p.groups + g);
      const float2 s = p.seg_sums[static_cast<int64_t>(tl.entry) * p.groups + g];
      s1[c] = s.x;
      s2[c] = s.y;
    });
    grad_rows<T, ACT, true>(p, Share(p, at, tl.begin, tl.end), mu, rs, af, s1, s2);
  }
}

// dw and db from the blocks' sums: 32 channels per block, every 32nd slot per
// warp, then the warps' sums in order.
__global__ void __launch_bounds__(1024) norm_params_kernel(const float* partial, int slots, int channels,
                                                          float* __restrict__ dw, float* __restrict__ db) {
  after_previous();
  __shared__ float part[32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int i = static_cast<int>(blockIdx.x) * 32 + lane;
  float s = 0.0f;
  if (i < 2 * channels) {
#pragma unroll 8
    for (int k = warp; k < slots; k += 32) s += partial[static_cast<int64_t>(k) * 2 * channels + i];
  }
  part[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || i >= 2 * channels) return;
  s = 0.0f;
  for (int k = 0; k < 32; ++k) s += part[k][lane];
  float* out = i < channels ? dw : db;
  if (out != nullptr) out[i < channels ? i : i - channels] = s;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct Plan {
  int32_t quads, team, threads, split, grid, tile_threads, tile_grid, merge_grid;
  int64_t loop_rows, tile_rows, max_long, max_tiles;
  bool longs;  // whether a segment can be too long for a team
};

int make_plan(const char* who, int64_t rows, int64_t channels, int64_t groups, int64_t nseg, int dtype, int activation,
              bool backward, Plan* pl) {
  const int64_t e = dtype == DGFX_F32 ? 4 : 2;
  if ((dtype != DGFX_F32 && dtype != DGFX_BF16) || rows < 0 || nseg < 0 || channels <= 0 || groups <= 0 ||
      channels % groups != 0 || channels * e % 16 != 0 || activation < DGFX_ACT_NONE ||
      activation > DGFX_ACT_SIGMOID) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, std::string(who) +
                                               ": need dtype fp32 or bf16, rows of a multiple of 16 bytes, groups that "
                                               "divide the channels, a known activation");
  }
  if (channels * e > 4096 || nseg >= (int64_t(1) << 31) || rows >= (int64_t(1) << 36)) {
    return fail(DGFX_ERR_UNSUPPORTED,
                std::string(who) + ": rows of at most 4096 bytes, fewer than 2^36 rows and 2^31 segments");
  }
  pl->quads = static_cast<int32_t>(channels / kCh);
  pl->split = channels / groups % kCh == 0 ? 1 : kCh;
  // A team grows while the average segment takes it more than four steps of
  // kAhead rows per thread, or more than two as long as the teams do not fill
  // the GPU: more threads for the same segment repeat the fixed work of its
  // sums (two or eight steps instead of four: within 1% over fifty drawn
  // sizes). It takes segments of up to eight steps; longer ones would hold up
  // their block. Where the teams do not fill the GPU, only of up to three:
  // row tiles spread over the SMs that are idle (36 segments of 331,464 rows in
  // all, 16 fp32 channels: 35 us instead of 50; at 300 segments of 250,001 rows,
  // which fill it, 404 us at six steps, 394 at eight). Only where 24 steps cover all
  // rows it takes any: three more launches would cost as much.
  const int ahead = (dtype == DGFX_F32 ? kAhead<float> : kAhead<__nv_bfloat16>) / 2;
  const int64_t average = nseg > 0 ? ceil_div(rows, nseg) : 1;
  auto step_rows = [&](int team) { return static_cast<int64_t>(team / pl->quads) * ahead; };
  int team = 32;
  while (team < 512 && (team < pl->quads || 4 * step_rows(team) < average ||
                        (nseg * team < kSms * 768 && 2 * step_rows(team) < average))) {
    team *= 2;
  }
  pl->team = team;
  pl->threads = std::max(team, 256);
  const int steps = nseg * team < kSms * 768 ? 3 : 8;
  pl->loop_rows = rows <= 24 * step_rows(team) ? rows : steps * step_rows(team);
  pl->longs = rows > pl->loop_rows;
  const int per_sm = (backward ? 3 : 4) * 256 / pl->threads;
  pl->grid = static_cast<int32_t>(
      std::max<int64_t>(1, std::min<int64_t>(ceil_div(nseg * team, pl->threads), kSms * per_sm)));
  if (nseg == 0) pl->grid = kSms;
  pl->tile_threads = pl->quads > 256 ? 512 : 256;
  pl->tile_grid = kSms * (backward ? 3 : 4) / (pl->tile_threads / 256);
  pl->tile_rows = std::max<int64_t>(2 * step_rows(team), ceil_div(rows, 2 * pl->tile_grid));  // two per block
  pl->max_long = rows / (pl->loop_rows + 1) + 1;
  pl->merge_grid = static_cast<int32_t>(std::min<int64_t>(pl->max_long * ceil_div(groups, 32), kSms * 4));
  pl->max_tiles = ceil_div(rows, pl->tile_rows) + pl->max_long;
  return DGFX_OK;
}

struct Work {
  unsigned long long* counter;
  longlong2* span;
  int32_t *seg, *base;
  float2 *tile_sums, *seg_sums;
  float* partial;
  size_t bytes;
  bool ok;
};

Work carve(void* ws, size_t cap, const Plan& pl, int64_t channels, int64_t groups, bool backward) {
  Arena a(ws, cap);
  Work w{};
  if (pl.longs) {
    w.counter = a.take<unsigned long long>(1);
    w.span = a.take<longlong2>(static_cast<size_t>(pl.max_long));
    w.seg = a.take<int32_t>(static_cast<size_t>(pl.max_long));
    w.base = a.take<int32_t>(static_cast<size_t>(pl.max_long));
    w.tile_sums = a.take<float2>(static_cast<size_t>(pl.max_tiles) * groups);
    if (backward) w.seg_sums = a.take<float2>(static_cast<size_t>(pl.max_long) * groups);
  }
  if (backward) w.partial = a.take<float>(static_cast<size_t>(pl.grid + (pl.longs ? pl.tile_grid : 0)) * 2 * channels);
  w.bytes = a.used;
  w.ok = a.ok();
  return w;
}

Params make_params(const Plan& pl, const Work& w, int64_t rows, int64_t channels, int64_t groups, int64_t nseg) {
  Params p{};
  p.rows = rows;
  p.nseg = nseg;
  p.channels = static_cast<int32_t>(channels);
  p.groups = static_cast<int32_t>(groups);
  p.quads = pl.quads;
  p.team = pl.team;
  p.split = pl.split;
  p.loop_rows = pl.loop_rows;
  p.tile_rows = pl.tile_rows;
  p.max_long = pl.max_long;
  p.max_tiles = pl.max_tiles;
  p.blocks_before = pl.grid;
  p.long_counter = w.counter;
  p.long_span = w.span;
  p.long_seg = w.seg;
  p.long_base = w.base;
  p.tile_sums = w.tile_sums;
  p.seg_sums = w.seg_sums;
  p.partial = w.partial;
  return p;
}

template <class T, int ACT>
void launch_forward(const Plan& pl, const Params& p, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(pl.threads / pl.team) * (pl.team * pl.split + p.groups) * sizeof(float);
  if (!pl.longs) {
    norm_forward_kernel<T, ACT><<<pl.grid, pl.threads, smem, stream>>>(p);
  } else {
    norm_list_kernel<<<1, 1024, 0, stream>>>(p);
    launch_after(norm_forward_kernel<T, ACT>, pl.grid, pl.threads, smem, stream, p);
    const size_t tsmem = (static_cast<size_t>(pl.tile_threads) * pl.split + p.groups) * sizeof(float);
    launch_after(norm_tile_stats_kernel<T>, pl.tile_grid, pl.tile_threads, tsmem, stream, p);
    launch_after(norm_merge_kernel<false>, pl.merge_grid, 256, 0, stream, p);
    launch_after(norm_tile_apply_kernel<T, ACT>, pl.tile_grid, pl.tile_threads, 0, stream, p);
  }
}

template <class T, int ACT>
void launch_backward(const Plan& pl, const Params& p, cudaStream_t stream) {
  const size_t sums = static_cast<size_t>(pl.threads / pl.team) * 2 * (pl.team * pl.split + p.groups) * sizeof(float);
  const size_t smem = std::max(sums, static_cast<size_t>(pl.threads) * 2 * kCh * sizeof(float));
  if (!pl.longs) {
    norm_backward_kernel<T, ACT><<<pl.grid, pl.threads, smem, stream>>>(p);
  } else {
    norm_list_kernel<<<1, 1024, 0, stream>>>(p);
    launch_after(norm_backward_kernel<T, ACT>, pl.grid, pl.threads, smem, stream, p);
    const size_t tsums = 2 * (static_cast<size_t>(pl.tile_threads) * pl.split + p.groups) * sizeof(float);
    const size_t tsmem = std::max(tsums, static_cast<size_t>(pl.tile_threads) * 2 * kCh * sizeof(float));
    launch_after(norm_tile_grad_kernel<T, ACT>, pl.tile_grid, pl.tile_threads, tsmem, stream, p);
    launch_after(norm_merge_kernel<true>, pl.merge_grid, 256, 0, stream, p);
    launch_after(norm_tile_grad_apply_kernel<T, ACT>, pl.tile_grid, pl.tile_threads, 0, stream, p);
  }
}

template <class T>
void run(int activation, bool backward, const Plan& pl, const Params& p, cudaStream_t stream) {
  switch (activation) {
    case DGFX_ACT_RELU:
      backward ? launch_backward<T, DGFX_ACT_RELU>(pl, p, stream) : launch_forward<T, DGFX_ACT_RELU>(pl, p, stream);
      break;
    case DGFX_ACT_SILU:
      backward ? launch_backward<T, DGFX_ACT_SILU>(pl, p, stream) : launch_forward<T, DGFX_ACT_SILU>(pl, p, stream);
      break;
    case DGFX_ACT_GELU:
      backward ? launch_backward<T, DGFX_ACT_GELU>(pl, p, stream) : launch_forward<T, DGFX_ACT_GELU>(pl, p, stream);
      break;
    case DGFX_ACT_SIGMOID:
      backward ? launch_backward<T, DGFX_ACT_SIGMOID>(pl, p, stream)
               : launch_forward<T, DGFX_ACT_SIGMOID>(pl, p, stream);
      break;
    default:
      backward ? launch_backward<T, DGFX_ACT_NONE>(pl, p, stream) : launch_forward<T, DGFX_ACT_NONE>(pl, p, stream);
      break;
  }
}

}  // namespace
}  // namespace dgfx

using namespace dgfx;

extern "C" int dgfx_segment_group_norm_workspace_size(int64_t rows, int64_t channels, int64_t groups, int64_t nseg,
                                                      int dtype, int32_t backward, size_t* bytes) {
  Plan pl;
  DGFX_TRY(make_plan("dgfx_segment_group_norm_workspace_size", rows, channels, groups, nseg, dtype, DGFX_ACT_NONE,
                     backward != 0, &pl));
  if (bytes == nullptr) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm_workspace_size: null result");
  }
  *bytes = carve(nullptr, 0, pl, channels, groups, backward != 0).bytes;
  return DGFX_OK;
}

extern "C" int dgfx_segment_group_norm(const void* d_x, int dtype, int64_t rows, int64_t channels, int64_t groups,
                                       const int64_t* d_offsets, int64_t nseg, const float* d_weight,
                                       const float* d_bias, float eps, int32_t activation, void* d_y, float* d_mean,
                                       float* d_rstd, void* d_workspace, size_t workspace_bytes, dgfx_stream stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  Plan pl;
  DGFX_TRY(make_plan("dgfx_segment_group_norm", rows, channels, groups, nseg, dtype, activation, false, &pl));
  if (d_offsets == nullptr || (rows > 0 && (d_x == nullptr || d_y == nullptr)) ||
      (nseg > 0 && (d_mean == nullptr || d_rstd == nullptr))) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm: null operand");
  }
  if (!ptr_aligned16(d_x) || !ptr_aligned16(d_y)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm: x and y must be 16-byte aligned");
  }
  if (!(eps > 0.0f)) return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm: eps must be positive");
  Work w{};
  if (pl.longs) {
    w = carve(d_workspace, workspace_bytes, pl, channels, groups, false);
    if (d_workspace == nullptr || !w.ok) return fail(DGFX_ERR_WORKSPACE, "dgfx_segment_group_norm: workspace too small");
    if (!ptr_aligned16(d_workspace)) {
      return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm: the workspace must be 16-byte aligned");
    }
  }
  Params p = make_params(pl, w, rows, channels, groups, nseg);
  p.x = d_x;
  p.off = d_offsets;
  p.weight = d_weight;
  p.bias = d_bias;
  p.y = d_y;
  p.mean = d_mean;
  p.rstd = d_rstd;
  p.eps = eps;
  if (dtype == DGFX_F32) run<float>(activation, false, pl, p, stream);
  else run<__nv_bfloat16>(activation, false, pl, p, stream);
  DGFX_CUDA_TRY(cudaGetLastError());
  return DGFX_OK;
}

extern "C" int dgfx_segment_group_norm_backward(const void* d_dy, const void* d_x, int dtype, int64_t rows,
                                                int64_t channels, int64_t groups, const int64_t* d_offsets,
                                                int64_t nseg, const float* d_mean, const float* d_rstd,
                                                const float* d_weight, const float* d_bias, int32_t activation,
                                                void* d_dx, float* d_dweight, float* d_dbias, void* d_workspace,
                                                size_t workspace_bytes, dgfx_stream stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  Plan pl;
  DGFX_TRY(make_plan("dgfx_segment_group_norm_backward", rows, channels, groups, nseg, dtype, activation, true, &pl));
  if (d_offsets == nullptr || (rows > 0 && (d_x == nullptr || d_dy == nullptr || d_dx == nullptr)) ||
      (nseg > 0 && (d_mean == nullptr || d_rstd == nullptr))) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm_backward: null operand");
  }
  if (!ptr_aligned16(d_x) || !ptr_aligned16(d_dy) || !ptr_aligned16(d_dx)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm_backward: operands must be 16-byte aligned");
  }
  const Work w = carve(d_workspace, workspace_bytes, pl, channels, groups, true);
  if (d_workspace == nullptr || !w.ok) {
    return fail(DGFX_ERR_WORKSPACE, "dgfx_segment_group_norm_backward: workspace too small");
  }
  if (!ptr_aligned16(d_workspace)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm_backward: the workspace must be 16-byte aligned");
  }
  Params p = make_params(pl, w, rows, channels, groups, nseg);
  p.x = d_x;
  p.dy = d_dy;
  p.off = d_offsets;
  p.weight = d_weight;
  p.bias = d_bias;
  p.y = d_dx;
  p.mean = const_cast<float*>(d_mean);
  p.rstd = const_cast<float*>(d_rstd);
  if (dtype == DGFX_F32) run<float>(activation, true, pl, p, stream);
  else run<__nv_bfloat16>(activation, true, pl, p, stream);
  DGFX_CUDA_TRY(cudaGetLastError());
  if (d_dweight != nullptr || d_dbias != nullptr) {
    launch_after(norm_params_kernel, static_cast<unsigned>(ceil_div(2 * channels, 32)), 1024, 0, stream, w.partial,
                 pl.grid + (pl.longs ? pl.tile_grid : 0), channels, d_dweight, d_dbias);
    DGFX_CUDA_TRY(cudaGetLastError());
  }
  return DGFX_OK;
}
