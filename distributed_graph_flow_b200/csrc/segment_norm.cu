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
// Bound by HBM. Short segments (a sampled graph) are read once: a team of
// threads holds the whole segment in registers, 32 KB per 256 threads, takes
// the sums and writes the result. A team is the smallest power of two of
// threads (32 .. 512, at least a row) that holds twice the average segment,
// so many small segments share a block. Longer segments are listed (in row
// order) and go through two more kernels: the first reads row tiles and
// leaves a mean and a centred sum of squares per tile and group, which the
// block that finishes a segment's last tile merges; the second applies them,
// tiles in reverse order, so that what the first read last is still in L2.
// When no segment can be long (all rows fit a team) only the first kernel is launched.
//
// Thread t of a team holds the quad (4 channels) t mod Q of every (team / Q)-th
// row, Q = C / 4: loads are whole rows and a thread's channels never change,
// so weights and the sums for dw and db stay in registers. Squares are summed
// around a mean (two passes over registers, or pairwise merges of means and
// centred squares along the rows of a tile), never as sum x^2 - mean^2. All sums are
// fp32 in an order fixed by the sizes: results do not change from run to
// run. Rows outside [off[0], off[nseg]) are written as zeros and their inputs
// are never used.
#include <algorithm>
#include <string>

#include "layer_math.cuh"

namespace dgfx {
namespace {

constexpr int kSms = 148;
constexpr int kCh = 4;

// Rows of a segment one thread holds (quads of bf16 take half the registers).
template <class T>
constexpr int kHold = sizeof(T) == 2 ? 16 : 8;

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
  // (count << 32 | tiles), blocks done with the short ones, a slot per
  // possible first row, the list (number, first tile), finished tiles, per
  // tile and group two sums.
  unsigned long long* long_counter;
  unsigned int* blocks_done;
  int32_t* long_slot;
  int32_t* long_seg;
  int32_t* long_base;
  int32_t* long_done;
  float2* tile_sums;
  float2* seg_sums;  // backward: S1 / n and S2 / n per long segment and group
  int64_t rows, nseg;
  int64_t hold_rows;  // rows a team holds in registers
  int64_t tile_rows;
  int64_t max_long, max_tiles;  // room of the list and of tile_sums
  int32_t channels, groups, quads;
  int32_t team;       // threads per team of the short-segment kernels
  int32_t split;      // values a thread gives to the group sums: 1 if a quad lies in one group, else 4
  int32_t blocks_before;  // backward: partial slots of the short-segment kernel
  float eps;
};

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

template <class T>
__device__ __forceinline__ typename Quad<T>::raw load_quad(const Params& p, const void* base, int64_t row, int col) {
  return __ldg(static_cast<const typename Quad<T>::raw*>(base) + row * p.quads + col);
}

template <class T>
__device__ __forceinline__ void store_quad(const Params& p, int64_t row, int col, const float (&f)[kCh]) {
  static_cast<typename Quad<T>::raw*>(p.y)[row * p.quads + col] = Quad<T>::pack(f);
}

// The affine parameters of this thread's channels.
struct Affine {
  float w[kCh], b[kCh];
  __device__ Affine(const Params& p, const Place& at) {
#pragma unroll
    for (int c = 0; c < kCh; ++c) {
      const int ch = at.col * kCh + c;
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

// Zeros in the rows outside of every segment.
template <class T>
__device__ __forceinline__ void zero_outside(const Params& p, int64_t lo, int64_t hi) {
  auto* y = static_cast<typename Quad<T>::raw*>(p.y);
  const int64_t threads = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t i = t; i < lo * p.quads; i += threads) y[i] = Quad<T>::zero();
  for (int64_t i = hi * p.quads + t; i < p.rows * p.quads; i += threads) y[i] = Quad<T>::zero();
}

// A long segment notes itself in the slot of its first row: segments of more
// than hold_rows rows begin at least that far apart, so no two share a slot.
__device__ __forceinline__ void note_long(const Params& p, int64_t s, int64_t begin) {
  p.long_slot[begin / (p.hold_rows + 1)] = static_cast<int32_t>(s) + 1;
}

// The last block of a short-segment kernel to get here turns the slots into
// the list of long segments, in row order (whatever order the teams ran in),
// with each one's first tile. Every thread of every block calls it.
__device__ __forceinline__ void list_longs(const Params& p, int64_t lo, int64_t hi, float* smem) {
  __shared__ int last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(p.blocks_done, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  const int64_t each = (p.max_long + blockDim.x - 1) / blockDim.x;
  const int64_t from = each * threadIdx.x, to = from + each < p.max_long ? from + each : p.max_long;
  auto tiles_of = [&](int64_t s) {
    const int64_t b = clamp64(p.off[s], lo, hi), e = clamp64(p.off[s + 1], b, hi);
    return static_cast<unsigned long long>((e - b + p.tile_rows - 1) / p.tile_rows);
  };
  unsigned long long mine = 0, all = 0;  // count << 32 | tiles
  for (int64_t i = from; i < to; ++i) {
    const int32_t s = __ldcg(p.long_slot + i);
    if (s != 0) mine += (1ull << 32) | tiles_of(s - 1);
  }
  unsigned long long at = block_exclusive_scan(mine, reinterpret_cast<unsigned long long*>(smem), &all);
  for (int64_t i = from; i < to; ++i) {
    const int32_t s = __ldcg(p.long_slot + i);
    if (s == 0) continue;
    const int64_t base = static_cast<int64_t>(at & 0xffffffffull);
    p.long_seg[at >> 32] = s - 1;
    // Ascending offsets fit; others stay inside of the tables.
    p.long_base[at >> 32] = static_cast<int32_t>(base < p.max_tiles ? base : p.max_tiles);
    at += (1ull << 32) | tiles_of(s - 1);
  }
  if (threadIdx.x == 0) *p.long_counter = all;
}

struct LongList {
  int count, tiles;
  __device__ explicit LongList(const Params& p) {
    const unsigned long long c = *p.long_counter;
    const int64_t t = static_cast<int64_t>(c & 0xffffffffull);
    count = static_cast<int>(c >> 32);
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
    const bool le = q < hi && __ldg(base + q) <= tile;
    const int k = 31 - __clz(static_cast<int>(__ballot_sync(0xffffffffu, le)));
    hi = min(hi, lo + step * (k + 1));
    lo = lo + step * k;
  }
  return lo;
}

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
template <class T, int ACT>
__global__ void __launch_bounds__(512, 2) norm_forward_kernel(Params p) {
  using Q = Quad<T>;
  constexpr int U = kHold<T>;
  extern __shared__ float smem[];
  const int in_block = threadIdx.x / p.team, t = threadIdx.x - in_block * p.team, bar = 1 + in_block;
  const Place at(p, t, p.team);
  const int g0 = at.col * kCh / (p.channels / p.groups);
  float* red = smem + in_block * (p.team * p.split + p.groups);
  float* gsum = red + p.team * p.split;
  const int64_t lo = clamp64(p.off[0], 0, p.rows), hi = clamp64(p.off[p.nseg], lo, p.rows);
  zero_outside<T>(p, lo, hi);
  const int cg = p.channels / p.groups;
  const int teams = blockDim.x / p.team;
  for (int64_t s = static_cast<int64_t>(blockIdx.x) * teams + in_block; s < p.nseg;
       s += static_cast<int64_t>(gridDim.x) * teams) {
    const int64_t begin = clamp64(p.off[s], lo, hi), end = clamp64(p.off[s + 1], begin, hi);
    if (end - begin > p.hold_rows) {
      if (t == 0) note_long(p, s, begin);
      continue;
    }
    const int n = static_cast<int>(end - begin);
    // This thread's rows: begin + rl + u per_pass for u < mine.
    const int mine = at.on && n > at.rl ? (n - at.rl + at.per_pass - 1) / at.per_pass : 0;
    const int step = at.per_pass * p.quads;
    const int64_t at0 = (begin + at.rl) * p.quads + at.col;
    const typename Q::raw* px = static_cast<const typename Q::raw*>(p.x) + at0;
    typename Q::raw v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = u < mine ? __ldg(px + u * step) : Q::zero();
    const float inv = n > 0 ? 1.0f / (static_cast<float>(n) * static_cast<float>(cg)) : 0.0f;
    float acc[1][kCh] = {};
#pragma unroll
    for (int u = 0; u < U; ++u) {  // rows past the end hold zeros
      float f[kCh];
      Q::unpack(v[u], f);
#pragma unroll
      for (int c = 0; c < kCh; ++c) acc[0][c] += f[c];
    }
    group_sums<1>(p, acc, at, t, p.team, bar, red, gsum);
    float mu[kCh];
    each_group(p, at, g0, [&](int c, int g) {
      mu[c] = at.on ? gsum[g] * inv : 0.0f;
      acc[0][c] = 0.0f;
    });
    for (int g = t; g < p.groups; g += p.team) p.mean[s * p.groups + g] = gsum[g] * inv;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u < mine) {
        float f[kCh];
        Q::unpack(v[u], f);
#pragma unroll
        for (int c = 0; c < kCh; ++c) acc[0][c] += (f[c] - mu[c]) * (f[c] - mu[c]);
      }
    }
    // Its first barrier also ends the reads of gsum above.
    group_sums<1>(p, acc, at, t, p.team, bar, red, gsum);
    float rs[kCh];
    each_group(p, at, g0, [&](int c, int g) { rs[c] = at.on ? rsqrtf(gsum[g] * inv + p.eps) : 0.0f; });
    for (int g = t; g < p.groups; g += p.team) p.rstd[s * p.groups + g] = rsqrtf(gsum[g] * inv + p.eps);
    if (mine > 0) {
      const Affine af(p, at);
      typename Q::raw* py = static_cast<typename Q::raw*>(p.y) + at0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u < mine) {
          float f[kCh];
          Q::unpack(v[u], f);
#pragma unroll
          for (int c = 0; c < kCh; ++c) f[c] = act_f<ACT>((f[c] - mu[c]) * rs[c] * af.w[c] + af.b[c]);
          py[u * step] = Q::pack(f);
        }
      }
    }
  }
  if (p.long_counter != nullptr) list_longs(p, lo, hi, smem);
}

// One row tile of a listed segment.
struct Tile {
  int entry, count_tiles, first;
  int64_t seg, begin, end, rows_of_seg;  // rows [begin, end)
  __device__ Tile(const Params& p, const LongList& all, int tile) {
    entry = find_long(p.long_base, all.count, tile);
    first = __ldg(p.long_base + entry);
    count_tiles = (entry + 1 < all.count ? __ldg(p.long_base + entry + 1) : all.tiles) - first;
    seg = __ldg(p.long_seg + entry);
    const int64_t lo = clamp64(p.off[0], 0, p.rows), hi = clamp64(p.off[p.nseg], lo, p.rows);
    const int64_t b = clamp64(p.off[seg], lo, hi), e = clamp64(p.off[seg + 1], b, hi);
    rows_of_seg = e - b;
    begin = b + static_cast<int64_t>(tile - first) * p.tile_rows;
    end = begin + p.tile_rows < e ? begin + p.tile_rows : e;
  }
};

// True for the whole block when this was the last of the segment's tiles; all
// tiles' sums are then visible to it.
__device__ __forceinline__ bool last_tile(const Params& p, const Tile& tile, int* flag) {
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) *flag = atomicAdd(p.long_done + tile.entry, 1) == tile.count_tiles - 1;
  __syncthreads();
  const bool last = *flag != 0;
  if (last) __threadfence();
  return last;
}

template <class T>
__global__ void __maxnreg__(64) norm_tile_stats_kernel(Params p) {
  using Q = Quad<T>;
  constexpr int B = 4;  // rows loaded at a time
  extern __shared__ float smem[];
  __shared__ int flag;
  float* red = smem;
  float* gsum = red + blockDim.x * p.split;
  const int threads = blockDim.x;
  const Place at(p, threadIdx.x, threads);
  const int g0 = at.col * kCh / (p.channels / p.groups);
  const LongList all(p);
  const int cg = p.channels / p.groups;
  for (int tile = blockIdx.x; tile < all.tiles; tile += gridDim.x) {
    const Tile tl(p, all, tile);
    // Mean and centred squares of this thread's rows, merged B rows at a time
    // (Chan, Golub and LeVeque, "Updating formulae and a pairwise algorithm
    // for computing sample variances", 1979).
    float mean[kCh] = {}, m2[kCh] = {}, have = 0.0f;
    if (at.on) {
      const int64_t step = at.per_pass;
      for (int64_t r = tl.begin + at.rl; r < tl.end; r += B * step) {
        typename Q::raw v[B];
        int k = 0;
#pragma unroll
        for (int i = 0; i < B; ++i) {
          if (r + i * step < tl.end) {
            v[i] = load_quad<T>(p, p.x, r + i * step, at.col);
            ++k;
          } else {
            v[i] = Q::zero();
          }
        }
        const float kf = static_cast<float>(k);
        const float ik = k == B ? 1.0f / B : 1.0f / kf;
        const float all = have + kf, share = kf / all;
        float sum[kCh] = {}, sq[kCh] = {}, f[B][kCh];
#pragma unroll
        for (int i = 0; i < B; ++i) {
          Q::unpack(v[i], f[i]);
#pragma unroll
          for (int c = 0; c < kCh; ++c) sum[c] += f[i][c];
        }
#pragma unroll
        for (int c = 0; c < kCh; ++c) sum[c] *= ik;
#pragma unroll
        for (int i = 0; i < B; ++i) {
          if (i < k) {
#pragma unroll
            for (int c = 0; c < kCh; ++c) sq[c] += (f[i][c] - sum[c]) * (f[i][c] - sum[c]);
          }
        }
#pragma unroll
        for (int c = 0; c < kCh; ++c) {
          const float d = sum[c] - mean[c];
          mean[c] += d * share;
          m2[c] += sq[c] + d * d * (have * share);
        }
        have = all;
      }
    }
    const float n_tile = static_cast<float>(tl.end - tl.begin) * static_cast<float>(cg);
    float acc[1][kCh];
#pragma unroll
    for (int c = 0; c < kCh; ++c) acc[0][c] = have * mean[c];
    group_sums<1>(p, acc, at, threadIdx.x, threads, 1, red, gsum);
    each_group(p, at, g0, [&](int c, int g) {
      const float d = at.on ? mean[c] - gsum[g] / n_tile : 0.0f;
      acc[0][c] = m2[c] + have * d * d;
    });
    for (int g = threadIdx.x; g < p.groups; g += threads) {
      p.tile_sums[static_cast<int64_t>(tile) * p.groups + g].x = gsum[g] / n_tile;
    }
    group_sums<1>(p, acc, at, threadIdx.x, threads, 1, red, gsum);
    for (int g = threadIdx.x; g < p.groups; g += threads) {
      p.tile_sums[static_cast<int64_t>(tile) * p.groups + g].y = gsum[g];
    }
    if (last_tile(p, tl, &flag)) {
      // Merge the segment's tiles, a warp per group.
      const int lane = threadIdx.x & 31;
      const float n_all = static_cast<float>(tl.rows_of_seg) * static_cast<float>(cg);
      const float n_full = static_cast<float>(p.tile_rows) * static_cast<float>(cg);
      const float n_last = static_cast<float>(tl.rows_of_seg - (tl.count_tiles - 1) * p.tile_rows) * static_cast<float>(cg);
      for (int g = threadIdx.x >> 5; g < p.groups; g += threads >> 5) {
        const float2* sums = p.tile_sums + static_cast<int64_t>(tl.first) * p.groups + g;
        float m = 0.0f;
        for (int k = lane; k < tl.count_tiles; k += 32) {
          m += (k == tl.count_tiles - 1 ? n_last : n_full) * __ldcg(&sums[static_cast<int64_t>(k) * p.groups].x);
        }
        m = warp_reduce_sum(m) / n_all;
        float q = 0.0f;
        for (int k = lane; k < tl.count_tiles; k += 32) {
          const float2 s = __ldcg(&sums[static_cast<int64_t>(k) * p.groups]);
          q += s.y + (k == tl.count_tiles - 1 ? n_last : n_full) * (s.x - m) * (s.x - m);
        }
        q = warp_reduce_sum(q) / n_all;
        if (lane == 0) {
          p.mean[tl.seg * p.groups + g] = m;
          p.rstd[tl.seg * p.groups + g] = rsqrtf(q + p.eps);
        }
      }
    }
    __syncthreads();
  }
}

template <class T, int ACT>
__global__ void __maxnreg__(64) norm_tile_apply_kernel(Params p) {
  using Q = Quad<T>;
  constexpr int B = 8;
  const Place at(p, threadIdx.x, blockDim.x);
  const int g0 = at.col * kCh / (p.channels / p.groups);
  const Affine af(p, at);
  const LongList all(p);
  for (int tile = all.tiles - 1 - static_cast<int>(blockIdx.x); tile >= 0; tile -= gridDim.x) {
    const Tile tl(p, all, tile);
    if (!at.on) continue;
    float mu[kCh], rs[kCh];
    each_group(p, at, g0, [&](int c, int g) {
      mu[c] = __ldg(p.mean + tl.seg * p.groups + g);
      rs[c] = __ldg(p.rstd + tl.seg * p.groups + g);
    });
    const int64_t step = at.per_pass;
    for (int64_t r = tl.begin + at.rl; r < tl.end; r += B * step) {
      typename Q::raw v[B];
#pragma unroll
      for (int i = 0; i < B; ++i) {
        v[i] = Q::zero();
        if (r + i * step < tl.end) v[i] = load_quad<T>(p, p.x, r + i * step, at.col);
      }
#pragma unroll
      for (int i = 0; i < B; ++i) {
        if (r + i * step < tl.end) {
          float f[kCh];
          Q::unpack(v[i], f);
#pragma unroll
          for (int c = 0; c < kCh; ++c) f[c] = act_f<ACT>((f[c] - mu[c]) * rs[c] * af.w[c] + af.b[c]);
          store_quad<T>(p, r + i * step, at.col, f);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------
// xhat, and w dz rounded before any subtraction, the same value in the sums
// and in dx: a segment of one value then cancels to zero exactly.
template <int ACT>
__device__ __forceinline__ void grad_terms(float x, float dy, float mu, float rs, float w, float b, float* xhat,
                                           float* dz, float* wdz) {
  *xhat = (x - mu) * rs;
  float v, slope;
  act_both_f<ACT>(*xhat * w + b, &v, &slope);
  *dz = __fmul_rn(dy, slope);
  *wdz = __fmul_rn(*dz, w);
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

template <class T, int ACT>
__global__ void __launch_bounds__(512, 1) norm_backward_kernel(Params p) {
  using Q = Quad<T>;
  constexpr int U = kHold<T>;
  extern __shared__ float smem[];
  const int in_block = threadIdx.x / p.team, t = threadIdx.x - in_block * p.team, bar = 1 + in_block;
  const Place at(p, t, p.team);
  const int g0 = at.col * kCh / (p.channels / p.groups);
  float* red = smem + in_block * 2 * (p.team * p.split + p.groups);
  float* gsum = red + 2 * p.team * p.split;
  const int64_t lo = clamp64(p.off[0], 0, p.rows), hi = clamp64(p.off[p.nseg], lo, p.rows);
  zero_outside<T>(p, lo, hi);
  const Affine af(p, at);
  const int cg = p.channels / p.groups;
  const int teams = blockDim.x / p.team;
  float dwb[2][kCh] = {};
  for (int64_t s = static_cast<int64_t>(blockIdx.x) * teams + in_block; s < p.nseg;
       s += static_cast<int64_t>(gridDim.x) * teams) {
    const int64_t begin = clamp64(p.off[s], lo, hi), end = clamp64(p.off[s + 1], begin, hi);
    if (begin == end) continue;
    if (end - begin > p.hold_rows) {
      if (t == 0) note_long(p, s, begin);
      continue;
    }
    const int n = static_cast<int>(end - begin);
    const int mine = at.on && n > at.rl ? (n - at.rl + at.per_pass - 1) / at.per_pass : 0;
    const int step = at.per_pass * p.quads;
    const int64_t at0 = (begin + at.rl) * p.quads + at.col;
    const typename Q::raw* px = static_cast<const typename Q::raw*>(p.x) + at0;
    const typename Q::raw* pd = static_cast<const typename Q::raw*>(p.dy) + at0;
    typename Q::raw v[U], d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = u < mine ? __ldg(px + u * step) : Q::zero();
      d[u] = u < mine ? __ldg(pd + u * step) : Q::zero();
    }
    const float inv = 1.0f / (static_cast<float>(n) * static_cast<float>(cg));
    float mu[kCh], rs[kCh], acc[2][kCh] = {};
    each_group(p, at, g0, [&](int c, int g) {
      mu[c] = at.on ? __ldg(p.mean + s * p.groups + g) : 0.0f;
      rs[c] = at.on ? __ldg(p.rstd + s * p.groups + g) : 0.0f;
    });
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u < mine) {
        float f[kCh], g[kCh];
        Q::unpack(v[u], f);
        Q::unpack(d[u], g);
#pragma unroll
        for (int c = 0; c < kCh; ++c) {
          float xh, dz, wdz;
          grad_terms<ACT>(f[c], g[c], mu[c], rs[c], af.w[c], af.b[c], &xh, &dz, &wdz);
          dwb[0][c] += dz * xh;
          dwb[1][c] += dz;
          acc[0][c] += wdz;
          acc[1][c] += wdz * xh;
        }
      }
    }
    group_sums<2>(p, acc, at, t, p.team, bar, red, gsum);
    if (mine > 0) {
      float s1[kCh], s2[kCh];
      typename Q::raw* py = static_cast<typename Q::raw*>(p.y) + at0;
      each_group(p, at, g0, [&](int c, int g) {
        s1[c] = gsum[g] * inv;
        s2[c] = gsum[p.groups + g] * inv;
      });
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u < mine) {
          float f[kCh], g[kCh];
          Q::unpack(v[u], f);
          Q::unpack(d[u], g);
#pragma unroll
          for (int c = 0; c < kCh; ++c) {
            float xh, dz, wdz;
            grad_terms<ACT>(f[c], g[c], mu[c], rs[c], af.w[c], af.b[c], &xh, &dz, &wdz);
            f[c] = rs[c] * (wdz - s1[c] - xh * s2[c]);
          }
          py[u * step] = Q::pack(f);
        }
      }
    }
  }
  write_partial(p, dwb, at, teams, in_block, smem, blockIdx.x);
  if (p.long_counter != nullptr) {
    __syncthreads();
    list_longs(p, lo, hi, smem);
  }
}

template <class T, int ACT>
__global__ void __maxnreg__(80) norm_tile_grad_kernel(Params p) {
  using Q = Quad<T>;
  constexpr int B = 4;
  extern __shared__ float smem[];
  __shared__ int flag;
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
    if (at.on) {
      float dwt[2][kCh] = {};  // this tile's, so that long sums stay pairwise
      const int64_t step = at.per_pass;
      for (int64_t r = tl.begin + at.rl; r < tl.end; r += B * step) {
        typename Q::raw v[B], d[B];
#pragma unroll
        for (int i = 0; i < B; ++i) {
          v[i] = Q::zero();
          d[i] = Q::zero();
          if (r + i * step < tl.end) {
            v[i] = load_quad<T>(p, p.x, r + i * step, at.col);
            d[i] = load_quad<T>(p, p.dy, r + i * step, at.col);
          }
        }
#pragma unroll
        for (int i = 0; i < B; ++i) {
          if (r + i * step < tl.end) {
            float f[kCh], g[kCh];
            Q::unpack(v[i], f);
            Q::unpack(d[i], g);
#pragma unroll
            for (int c = 0; c < kCh; ++c) {
              float xh, dz, wdz;
              grad_terms<ACT>(f[c], g[c], mu[c], rs[c], af.w[c], af.b[c], &xh, &dz, &wdz);
              dwt[0][c] += dz * xh;
              dwt[1][c] += dz;
              acc[0][c] += wdz;
              acc[1][c] += wdz * xh;
            }
          }
        }
      }
#pragma unroll
      for (int c = 0; c < kCh; ++c) {
        dwb[0][c] += dwt[0][c];
        dwb[1][c] += dwt[1][c];
      }
    }
    group_sums<2>(p, acc, at, threadIdx.x, threads, 1, red, gsum);
    for (int g = threadIdx.x; g < p.groups; g += threads) {
      p.tile_sums[static_cast<int64_t>(tile) * p.groups + g] = make_float2(gsum[g], gsum[p.groups + g]);
    }
    if (last_tile(p, tl, &flag)) {
      const int lane = threadIdx.x & 31;
      const float n_all = static_cast<float>(tl.rows_of_seg) * static_cast<float>(cg);
      for (int g = threadIdx.x >> 5; g < p.groups; g += threads >> 5) {
        const float2* sums = p.tile_sums + static_cast<int64_t>(tl.first) * p.groups + g;
        float a = 0.0f, b = 0.0f;
        for (int k = lane; k < tl.count_tiles; k += 32) {
          const float2 s = __ldcg(&sums[static_cast<int64_t>(k) * p.groups]);
          a += s.x;
          b += s.y;
        }
        a = warp_reduce_sum(a) / n_all;
        b = warp_reduce_sum(b) / n_all;
        if (lane == 0) p.seg_sums[static_cast<int64_t>(tl.entry) * p.groups + g] = make_float2(a, b);
      }
    }
    __syncthreads();
  }
  write_partial(p, dwb, at, 1, 0, smem, p.blocks_before + blockIdx.x);
}

template <class T, int ACT>
__global__ void __maxnreg__(80) norm_tile_grad_apply_kernel(Params p) {
  using Q = Quad<T>;
  constexpr int B = 4;
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
      const float2 s = __ldg(p.seg_sums + static_cast<int64_t>(tl.entry) * p.groups + g);
      s1[c] = s.x;
      s2[c] = s.y;
    });
    const int64_t step = at.per_pass;
    for (int64_t r = tl.begin + at.rl; r < tl.end; r += B * step) {
      typename Q::raw v[B], d[B];
#pragma unroll
      for (int i = 0; i < B; ++i) {
        v[i] = Q::zero();
        d[i] = Q::zero();
        if (r + i * step < tl.end) {
          v[i] = load_quad<T>(p, p.x, r + i * step, at.col);
          d[i] = load_quad<T>(p, p.dy, r + i * step, at.col);
        }
      }
#pragma unroll
      for (int i = 0; i < B; ++i) {
        if (r + i * step < tl.end) {
          float f[kCh], g[kCh];
          Q::unpack(v[i], f);
          Q::unpack(d[i], g);
#pragma unroll
          for (int c = 0; c < kCh; ++c) {
            float xh, dz, wdz;
            grad_terms<ACT>(f[c], g[c], mu[c], rs[c], af.w[c], af.b[c], &xh, &dz, &wdz);
            f[c] = rs[c] * (wdz - s1[c] - xh * s2[c]);
          }
          store_quad<T>(p, r + i * step, at.col, f);
        }
      }
    }
  }
}

// dw and db from the blocks' sums: 32 channels per block, every eighth slot
// per warp, then the warps' sums in order.
__global__ void __launch_bounds__(256) norm_params_kernel(const float* __restrict__ partial, int slots, int channels,
                                                          float* __restrict__ dw, float* __restrict__ db) {
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int i = static_cast<int>(blockIdx.x) * 32 + lane;
  float s = 0.0f;
  if (i < 2 * channels) {
#pragma unroll 8
    for (int k = warp; k < slots; k += 8) s += __ldg(partial + static_cast<int64_t>(k) * 2 * channels + i);
  }
  part[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || i >= 2 * channels) return;
  s = 0.0f;
  for (int k = 0; k < 8; ++k) s += part[k][lane];
  float* out = i < channels ? dw : db;
  if (out != nullptr) out[i < channels ? i : i - channels] = s;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct Plan {
  int32_t quads, team, threads, split, grid, tile_threads, tile_grid;
  int64_t hold_rows, tile_rows, max_long, max_tiles;
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
  const int hold = dtype == DGFX_F32 ? kHold<float> : kHold<__nv_bfloat16>;
  pl->quads = static_cast<int32_t>(channels / kCh);
  pl->split = channels / groups % kCh == 0 ? 1 : kCh;
  const int64_t average = nseg > 0 ? ceil_div(rows, nseg) : 1;
  int team = 32;
  while (team < 512 && (team < pl->quads || static_cast<int64_t>(team / pl->quads) * hold < 2 * average)) team *= 2;
  pl->team = team;
  pl->threads = std::max(team, 256);
  pl->hold_rows = static_cast<int64_t>(team / pl->quads) * hold;
  pl->longs = rows > pl->hold_rows;
  const int per_sm = backward ? (pl->threads == 512 ? 1 : 2) : (pl->threads == 512 ? 2 : 4);
  pl->grid = static_cast<int32_t>(
      std::max<int64_t>(1, std::min<int64_t>(ceil_div(nseg * team, pl->threads), kSms * per_sm)));
  if (nseg == 0) pl->grid = kSms;
  pl->tile_threads = pl->quads > 256 ? 512 : 256;
  pl->tile_grid = kSms * (backward ? 3 : 4) / (pl->tile_threads / 256);
  pl->tile_rows = std::max<int64_t>(pl->hold_rows, ceil_div(rows, kSms * 16));
  pl->max_long = rows / (pl->hold_rows + 1) + 1;
  pl->max_tiles = ceil_div(rows, pl->tile_rows) + pl->max_long;
  return DGFX_OK;
}

struct Work {
  unsigned long long* counter;
  unsigned int* blocks;
  int32_t *slot, *seg, *base, *done;
  float2 *tile_sums, *seg_sums;
  float* partial;
  size_t clear_bytes, bytes;
  bool ok;
};

Work carve(void* ws, size_t cap, const Plan& pl, int64_t channels, int64_t groups, bool backward) {
  Arena a(ws, cap);
  Work w{};
  if (pl.longs) {
    // The counters and slots are cleared together.
    w.counter = a.take<unsigned long long>(1);
    w.blocks = a.take<unsigned int>(1);
    w.slot = a.take<int32_t>(static_cast<size_t>(pl.max_long));
    w.done = a.take<int32_t>(static_cast<size_t>(pl.max_long));
    w.clear_bytes = a.used;
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
  p.hold_rows = pl.hold_rows;
  p.tile_rows = pl.tile_rows;
  p.max_long = pl.max_long;
  p.max_tiles = pl.max_tiles;
  p.blocks_before = pl.grid;
  p.long_counter = w.counter;
  p.blocks_done = w.blocks;
  p.long_slot = w.slot;
  p.long_seg = w.seg;
  p.long_base = w.base;
  p.long_done = w.done;
  p.tile_sums = w.tile_sums;
  p.seg_sums = w.seg_sums;
  p.partial = w.partial;
  return p;
}

template <class T, int ACT>
void launch_forward(const Plan& pl, const Params& p, cudaStream_t stream) {
  const size_t smem = static_cast<size_t>(pl.threads / pl.team) * (pl.team * pl.split + p.groups) * sizeof(float);
  norm_forward_kernel<T, ACT><<<pl.grid, pl.threads, smem, stream>>>(p);
  if (pl.longs) {
    const size_t tsmem = (static_cast<size_t>(pl.tile_threads) * pl.split + p.groups) * sizeof(float);
    norm_tile_stats_kernel<T><<<pl.tile_grid, pl.tile_threads, tsmem, stream>>>(p);
    norm_tile_apply_kernel<T, ACT><<<pl.tile_grid, pl.tile_threads, 0, stream>>>(p);
  }
}

template <class T, int ACT>
void launch_backward(const Plan& pl, const Params& p, cudaStream_t stream) {
  const size_t sums = static_cast<size_t>(pl.threads / pl.team) * 2 * (pl.team * pl.split + p.groups) * sizeof(float);
  const size_t smem = std::max(sums, static_cast<size_t>(pl.threads) * 2 * kCh * sizeof(float));
  norm_backward_kernel<T, ACT><<<pl.grid, pl.threads, smem, stream>>>(p);
  if (pl.longs) {
    const size_t tsums = 2 * (static_cast<size_t>(pl.tile_threads) * pl.split + p.groups) * sizeof(float);
    const size_t tsmem = std::max(tsums, static_cast<size_t>(pl.tile_threads) * 2 * kCh * sizeof(float));
    norm_tile_grad_kernel<T, ACT><<<pl.tile_grid, pl.tile_threads, tsmem, stream>>>(p);
    norm_tile_grad_apply_kernel<T, ACT><<<pl.tile_grid, pl.tile_threads, 0, stream>>>(p);
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
    DGFX_CUDA_TRY(cudaMemsetAsync(d_workspace, 0, w.clear_bytes, stream));
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
  if (pl.longs) DGFX_CUDA_TRY(cudaMemsetAsync(d_workspace, 0, w.clear_bytes, stream));
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
    norm_params_kernel<<<static_cast<unsigned>(ceil_div(2 * channels, 32)), 256, 0, stream>>>(
        w.partial, pl.grid + (pl.longs ? pl.tile_grid : 0), static_cast<int>(channels), d_dweight, d_dbias);
    DGFX_CUDA_TRY(cudaGetLastError());
  }
  return DGFX_OK;
}
