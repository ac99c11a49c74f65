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
// A block takes a segment at a time. Thread t holds the 16-byte column
// t mod V (V = vectors per row) of every (threads / V)-th row, so a block's loads are
// whole rows, and a thread's channels never change: weights and the sums for
// dw and db stay in registers. Squares are summed around the mean (two
// passes), never as sum x^2 - mean^2. All sums are fp32 in a fixed order:
// results do not change from run to run. Rows outside [off[0], off[nseg])
// are written as zeros and their inputs are never used.
#include <algorithm>
#include <string>

#include "layer_math.cuh"

namespace dgfx {
namespace {

struct Params {
  const void* x;
  const void* dy;
  const int64_t* off;
  const float* weight;
  const float* bias;
  void* y;  // output, or dx going backward
  float* mean;
  float* rstd;
  float* partial;  // [blocks, 2, C]: dw and db of one block
  int64_t rows, nseg;
  int32_t channels, groups, vecs, per_pass;  // per_pass: rows a block covers at a time
  float eps;
};

// Sums of acc[k][channel of this thread] over the block's rows and each
// group's channels: gsum[k * groups + g], for all threads after the call.
// red holds K * per_pass * C floats. Every thread of the block calls it.
template <int K, int N>
__device__ __forceinline__ void group_sums(const Params& p, const float (&acc)[K][N], bool on, int rl, int col, float* red,
                                           float* gsum) {
  const int C = p.channels;
  if (on) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int c = 0; c < N; ++c) red[(k * p.per_pass + rl) * C + col * N + c] = acc[k][c];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < K * C; i += blockDim.x) {
    const int k = i / C, c = i - k * C;
    float s = 0.0f;
    for (int r = 0; r < p.per_pass; ++r) s += red[(k * p.per_pass + r) * C + c];
    red[k * p.per_pass * C + c] = s;
  }
  __syncthreads();
  const int cg = C / p.groups;
  if (cg <= 32) {
    for (int i = threadIdx.x; i < K * p.groups; i += blockDim.x) {
      const int k = i / p.groups, g = i - k * p.groups;
      float s = 0.0f;
      for (int c = 0; c < cg; ++c) s += red[k * p.per_pass * C + g * cg + c];
      gsum[i] = s;
    }
  } else {
    const int lane = threadIdx.x & 31;
    for (int i = threadIdx.x >> 5; i < K * p.groups; i += blockDim.x >> 5) {
      const int k = i / p.groups, g = i - k * p.groups;
      float s = 0.0f;
      for (int c = lane; c < cg; c += 32) s += red[k * p.per_pass * C + g * cg + c];
      s = warp_reduce_sum(s);
      if (lane == 0) gsum[i] = s;
    }
  }
  __syncthreads();
}

// Zeros in the rows outside of every segment.
__device__ __forceinline__ void zero_outside(const Params& p, int64_t lo, int64_t hi) {
  uint4* y = static_cast<uint4*>(p.y);
  const int64_t threads = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t i = t; i < lo * p.vecs; i += threads) y[i] = make_uint4(0, 0, 0, 0);
  for (int64_t i = hi * p.vecs + t; i < p.rows * p.vecs; i += threads) y[i] = make_uint4(0, 0, 0, 0);
}

template <class T, int ACT>
__global__ void norm_forward_kernel(Params p) {
  constexpr int N = Vec16<T>::N;
  extern __shared__ float smem[];
  float* red = smem;
  float* gsum = red + p.per_pass * p.channels;
  float* gmean = gsum + p.groups;
  const int rl = threadIdx.x / p.vecs, col = threadIdx.x - rl * p.vecs;
  const bool on = rl < p.per_pass;
  const int cg = p.channels / p.groups;
  const uint4* x = static_cast<const uint4*>(p.x);
  uint4* y = static_cast<uint4*>(p.y);
  const int64_t lo = clamp64(p.off[0], 0, p.rows), hi = clamp64(p.off[p.nseg], lo, p.rows);
  zero_outside(p, lo, hi);
  float w[N], b[N];
  int grp[N];
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const int ch = on ? col * N + c : 0;
    w[c] = p.weight != nullptr ? p.weight[ch] : 1.0f;
    b[c] = p.bias != nullptr ? p.bias[ch] : 0.0f;
    grp[c] = ch / cg;
  }
  for (int64_t s = blockIdx.x; s < p.nseg; s += gridDim.x) {
    const int64_t begin = clamp64(p.off[s], lo, hi), end = clamp64(p.off[s + 1], begin, hi);
    const float inv = 1.0f / (static_cast<float>(end - begin) * static_cast<float>(cg));
    float acc[1][N];
#pragma unroll
    for (int c = 0; c < N; ++c) acc[0][c] = 0.0f;
    if (on) {
      for (int64_t r = begin + rl; r < end; r += p.per_pass) {
        float f[N];
        Vec16<T>::unpack(__ldg(x + r * p.vecs + col), f);
#pragma unroll
        for (int c = 0; c < N; ++c) acc[0][c] += f[c];
      }
    }
    group_sums<1, N>(p, acc, on, rl, col, red, gsum);
    float mu[N];
#pragma unroll
    for (int c = 0; c < N; ++c) {
      mu[c] = end > begin ? gsum[grp[c]] * inv : 0.0f;
      acc[0][c] = 0.0f;
    }
    for (int g = threadIdx.x; g < p.groups; g += blockDim.x) gmean[g] = end > begin ? gsum[g] * inv : 0.0f;
    if (on) {
      for (int64_t r = begin + rl; r < end; r += p.per_pass) {
        float f[N];
        Vec16<T>::unpack(__ldg(x + r * p.vecs + col), f);
#pragma unroll
        for (int c = 0; c < N; ++c) acc[0][c] += (f[c] - mu[c]) * (f[c] - mu[c]);
      }
    }
    __syncthreads();
    group_sums<1, N>(p, acc, on, rl, col, red, gsum);
    float rs[N];
#pragma unroll
    for (int c = 0; c < N; ++c) rs[c] = rsqrtf((end > begin ? gsum[grp[c]] * inv : 0.0f) + p.eps);
    for (int g = threadIdx.x; g < p.groups; g += blockDim.x) {
      p.mean[s * p.groups + g] = gmean[g];
      p.rstd[s * p.groups + g] = rsqrtf((end > begin ? gsum[g] * inv : 0.0f) + p.eps);
    }
    if (on) {
      for (int64_t r = begin + rl; r < end; r += p.per_pass) {
        float f[N];
        Vec16<T>::unpack(__ldg(x + r * p.vecs + col), f);
#pragma unroll
        for (int c = 0; c < N; ++c) f[c] = act_f<ACT>((f[c] - mu[c]) * rs[c] * w[c] + b[c]);
        y[r * p.vecs + col] = Vec16<T>::pack(f);
      }
    }
    __syncthreads();  // gsum and gmean are written again for the next segment
  }
}

template <class T, int ACT>
__global__ void norm_backward_kernel(Params p) {
  constexpr int N = Vec16<T>::N;
  extern __shared__ float smem[];
  float* red = smem;
  float* gsum = red + 2 * p.per_pass * p.channels;
  const int rl = threadIdx.x / p.vecs, col = threadIdx.x - rl * p.vecs;
  const bool on = rl < p.per_pass;
  const int cg = p.channels / p.groups;
  const uint4* x = static_cast<const uint4*>(p.x);
  const uint4* dy = static_cast<const uint4*>(p.dy);
  uint4* dx = static_cast<uint4*>(p.y);
  const int64_t lo = clamp64(p.off[0], 0, p.rows), hi = clamp64(p.off[p.nseg], lo, p.rows);
  zero_outside(p, lo, hi);
  float w[N], b[N], dwb[2][N];
  int grp[N];
#pragma unroll
  for (int c = 0; c < N; ++c) {
    const int ch = on ? col * N + c : 0;
    w[c] = p.weight != nullptr ? p.weight[ch] : 1.0f;
    b[c] = p.bias != nullptr ? p.bias[ch] : 0.0f;
    grp[c] = ch / cg;
    dwb[0][c] = dwb[1][c] = 0.0f;
  }
  for (int64_t s = blockIdx.x; s < p.nseg; s += gridDim.x) {
    const int64_t begin = clamp64(p.off[s], lo, hi), end = clamp64(p.off[s + 1], begin, hi);
    if (begin == end) continue;
    const float inv = 1.0f / (static_cast<float>(end - begin) * static_cast<float>(cg));
    float mu[N], rs[N], acc[2][N];
#pragma unroll
    for (int c = 0; c < N; ++c) {
      mu[c] = p.mean[s * p.groups + grp[c]];
      rs[c] = p.rstd[s * p.groups + grp[c]];
      acc[0][c] = acc[1][c] = 0.0f;
    }
    if (on) {
      for (int64_t r = begin + rl; r < end; r += p.per_pass) {
        float f[N], d[N];
        Vec16<T>::unpack(__ldg(x + r * p.vecs + col), f);
        Vec16<T>::unpack(__ldg(dy + r * p.vecs + col), d);
#pragma unroll
        for (int c = 0; c < N; ++c) {
          const float xh = (f[c] - mu[c]) * rs[c];
          float v, sl;
          act_both_f<ACT>(xh * w[c] + b[c], &v, &sl);
          const float dz = d[c] * sl;
          dwb[0][c] += dz * xh;
          dwb[1][c] += dz;
          acc[0][c] += __fmul_rn(dz, w[c]);
          acc[1][c] += __fmul_rn(dz, w[c]) * xh;
        }
      }
    }
    group_sums<2, N>(p, acc, on, rl, col, red, gsum);
    if (on) {
      float s1[N], s2[N];
#pragma unroll
      for (int c = 0; c < N; ++c) {
        s1[c] = gsum[grp[c]] * inv;
        s2[c] = gsum[p.groups + grp[c]] * inv;
      }
      for (int64_t r = begin + rl; r < end; r += p.per_pass) {
        float f[N], d[N];
        Vec16<T>::unpack(__ldg(x + r * p.vecs + col), f);
        Vec16<T>::unpack(__ldg(dy + r * p.vecs + col), d);
#pragma unroll
        for (int c = 0; c < N; ++c) {
          const float xh = (f[c] - mu[c]) * rs[c];
          float v, sl;
          act_both_f<ACT>(xh * w[c] + b[c], &v, &sl);
          // Rounded before the subtraction, as in the sums: a segment of one
          // value then cancels to zero exactly.
          const float g = __fmul_rn(d[c] * sl, w[c]);
          f[c] = rs[c] * (g - s1[c] - xh * s2[c]);
        }
        dx[r * p.vecs + col] = Vec16<T>::pack(f);
      }
    }
    __syncthreads();
  }
  // This block's sums for dw and db: over its row lanes, in order.
  __syncthreads();
  if (on) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int c = 0; c < N; ++c) red[(k * p.per_pass + rl) * p.channels + col * N + c] = dwb[k][c];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.channels; i += blockDim.x) {
    const int k = i / p.channels, c = i - k * p.channels;
    float s = 0.0f;
    for (int r = 0; r < p.per_pass; ++r) s += red[(k * p.per_pass + r) * p.channels + c];
    p.partial[(static_cast<int64_t>(blockIdx.x) * 2 + k) * p.channels + c] = s;
  }
}

// dw and db from the blocks' sums: one warp per channel and kind, each lane
// every 32nd block, then a fixed tree.
__global__ void norm_params_kernel(const float* __restrict__ partial, int blocks, int channels, float* __restrict__ dw,
                                   float* __restrict__ db) {
  const int lane = threadIdx.x & 31;
  const int i = static_cast<int>((static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5);
  if (i >= 2 * channels) return;
  float s = 0.0f;
  for (int k = lane; k < blocks; k += 32) s += partial[static_cast<int64_t>(k) * 2 * channels + i];
  s = warp_reduce_sum(s);
  if (lane != 0) return;
  if (i < channels) {
    if (dw != nullptr) dw[i] = s;
  } else if (db != nullptr) {
    db[i - channels] = s;
  }
}

struct Shape {
  int vecs, threads, per_pass;
};

int shape_of(const char* who, int64_t rows, int64_t channels, int64_t groups, int64_t nseg, int dtype, int activation,
             Shape* out) {
  const int64_t e = dtype == DGFX_F32 ? 4 : 2;
  if ((dtype != DGFX_F32 && dtype != DGFX_BF16) || rows < 0 || nseg < 0 || channels <= 0 || groups <= 0 ||
      channels % groups != 0 || channels * e % 16 != 0 || activation < DGFX_ACT_NONE ||
      activation > DGFX_ACT_SIGMOID) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, std::string(who) +
                                               ": need dtype fp32 or bf16, rows of a multiple of 16 bytes, groups that "
                                               "divide the channels, a known activation");
  }
  const int64_t vecs = channels * e / 16;
  if (vecs > 256 || nseg >= (int64_t(1) << 31)) {
    return fail(DGFX_ERR_UNSUPPORTED, std::string(who) + ": rows of at most 4096 bytes and fewer than 2^31 segments");
  }
  out->vecs = static_cast<int>(vecs);
  out->threads = 256;
  out->per_pass = out->threads / out->vecs;
  return DGFX_OK;
}

constexpr int kMaxBlocks = 148 * 4;

int blocks_for(int64_t nseg) { return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(nseg, kMaxBlocks))); }

template <class T>
void launch_forward(int activation, int grid, int threads, size_t smem, cudaStream_t stream, const Params& p) {
  switch (activation) {
    case DGFX_ACT_RELU: norm_forward_kernel<T, DGFX_ACT_RELU><<<grid, threads, smem, stream>>>(p); break;
    case DGFX_ACT_SILU: norm_forward_kernel<T, DGFX_ACT_SILU><<<grid, threads, smem, stream>>>(p); break;
    case DGFX_ACT_GELU: norm_forward_kernel<T, DGFX_ACT_GELU><<<grid, threads, smem, stream>>>(p); break;
    case DGFX_ACT_SIGMOID: norm_forward_kernel<T, DGFX_ACT_SIGMOID><<<grid, threads, smem, stream>>>(p); break;
    default: norm_forward_kernel<T, DGFX_ACT_NONE><<<grid, threads, smem, stream>>>(p); break;
  }
}

template <class T>
void launch_backward(int activation, int grid, int threads, size_t smem, cudaStream_t stream, const Params& p) {
  switch (activation) {
    case DGFX_ACT_RELU: norm_backward_kernel<T, DGFX_ACT_RELU><<<grid, threads, smem, stream>>>(p); break;
    case DGFX_ACT_SILU: norm_backward_kernel<T, DGFX_ACT_SILU><<<grid, threads, smem, stream>>>(p); break;
    case DGFX_ACT_GELU: norm_backward_kernel<T, DGFX_ACT_GELU><<<grid, threads, smem, stream>>>(p); break;
    case DGFX_ACT_SIGMOID: norm_backward_kernel<T, DGFX_ACT_SIGMOID><<<grid, threads, smem, stream>>>(p); break;
    default: norm_backward_kernel<T, DGFX_ACT_NONE><<<grid, threads, smem, stream>>>(p); break;
  }
}

}  // namespace
}  // namespace dgfx

using namespace dgfx;

extern "C" int dgfx_segment_group_norm_workspace_size(int64_t rows, int64_t channels, int64_t groups, int64_t nseg,
                                                      int dtype, int32_t backward, size_t* bytes) {
  Shape sh;
  DGFX_TRY(shape_of("dgfx_segment_group_norm_workspace_size", rows, channels, groups, nseg, dtype, DGFX_ACT_NONE, &sh));
  if (bytes == nullptr) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm_workspace_size: null result");
  }
  Arena arena(nullptr, 0);
  if (backward) arena.take<float>(static_cast<size_t>(kMaxBlocks) * 2 * channels);
  *bytes = arena.used;
  return DGFX_OK;
}

extern "C" int dgfx_segment_group_norm(const void* d_x, int dtype, int64_t rows, int64_t channels, int64_t groups,
                                       const int64_t* d_offsets, int64_t nseg, const float* d_weight,
                                       const float* d_bias, float eps, int32_t activation, void* d_y, float* d_mean,
                                       float* d_rstd, void* d_workspace, size_t workspace_bytes, dgfx_stream stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  Shape sh;
  DGFX_TRY(shape_of("dgfx_segment_group_norm", rows, channels, groups, nseg, dtype, activation, &sh));
  if (d_offsets == nullptr || (rows > 0 && (d_x == nullptr || d_y == nullptr)) ||
      (nseg > 0 && (d_mean == nullptr || d_rstd == nullptr))) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm: null operand");
  }
  if (!ptr_aligned16(d_x) || !ptr_aligned16(d_y)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm: x and y must be 16-byte aligned");
  }
  if (!(eps > 0.0f)) return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm: eps must be positive");
  (void)d_workspace;
  (void)workspace_bytes;
  Params p{};
  p.x = d_x;
  p.off = d_offsets;
  p.weight = d_weight;
  p.bias = d_bias;
  p.y = d_y;
  p.mean = d_mean;
  p.rstd = d_rstd;
  p.rows = rows;
  p.nseg = nseg;
  p.channels = static_cast<int32_t>(channels);
  p.groups = static_cast<int32_t>(groups);
  p.vecs = sh.vecs;
  p.per_pass = sh.per_pass;
  p.eps = eps;
  const int grid = nseg == 0 ? 148 : blocks_for(nseg);
  const size_t smem = (static_cast<size_t>(sh.per_pass) * channels + 2 * groups) * sizeof(float);
  if (dtype == DGFX_F32) launch_forward<float>(activation, grid, sh.threads, smem, stream, p);
  else launch_forward<__nv_bfloat16>(activation, grid, sh.threads, smem, stream, p);
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
  Shape sh;
  DGFX_TRY(shape_of("dgfx_segment_group_norm_backward", rows, channels, groups, nseg, dtype, activation, &sh));
  if (d_offsets == nullptr || (rows > 0 && (d_x == nullptr || d_dy == nullptr || d_dx == nullptr)) ||
      (nseg > 0 && (d_mean == nullptr || d_rstd == nullptr))) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm_backward: null operand");
  }
  if (!ptr_aligned16(d_x) || !ptr_aligned16(d_dy) || !ptr_aligned16(d_dx)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_segment_group_norm_backward: operands must be 16-byte aligned");
  }
  Arena arena(d_workspace, workspace_bytes);
  float* partial = arena.take<float>(static_cast<size_t>(kMaxBlocks) * 2 * channels);
  if (d_workspace == nullptr || !arena.ok()) {
    return fail(DGFX_ERR_WORKSPACE, "dgfx_segment_group_norm_backward: workspace too small");
  }
  Params p{};
  p.x = d_x;
  p.dy = d_dy;
  p.off = d_offsets;
  p.weight = d_weight;
  p.bias = d_bias;
  p.y = d_dx;
  p.mean = const_cast<float*>(d_mean);
  p.rstd = const_cast<float*>(d_rstd);
  p.partial = partial;
  p.rows = rows;
  p.nseg = nseg;
  p.channels = static_cast<int32_t>(channels);
  p.groups = static_cast<int32_t>(groups);
  p.vecs = sh.vecs;
  p.per_pass = sh.per_pass;
  const int grid = nseg == 0 ? 148 : blocks_for(nseg);
  const size_t smem = (2 * static_cast<size_t>(sh.per_pass) * channels + 2 * groups) * sizeof(float);
  if (dtype == DGFX_F32) launch_backward<float>(activation, grid, sh.threads, smem, stream, p);
  else launch_backward<__nv_bfloat16>(activation, grid, sh.threads, smem, stream, p);
  DGFX_CUDA_TRY(cudaGetLastError());
  norm_params_kernel<<<static_cast<unsigned>(ceil_div(2 * channels, 8)), 256, 0, stream>>>(
      partial, grid, static_cast<int>(channels), d_dweight, d_dbias);
  DGFX_CUDA_TRY(cudaGetLastError());
  return DGFX_OK;
}
