// Dense layer after neighbour aggregation on the 5th-generation tensor cores.
//
// Computes Y = act(concat[X1, X2] @ W^T + b) in bf16 with fp32 accumulation:
// the GraphSAGE / MPNN update "concat[x_dst, agg] -> Dense -> ReLU"
// (dgf/src/learning/jax/layers/hetero_gnn.py:302-312 with GenericBlock's
// nn.Dense, dgf/src/learning/jax/layers/standard.py:238-270). The concat is
// never materialised: the first k1/64 K-blocks of a tile come from X1's
// tensor map, the rest from X2's.
//
// Kernel structure (one persistent CTA per SM, 6 warps):
//   warp 0   TMA producer: per K-block a 128x64 tile of X1|X2 and a BNx64
//            tile of W (both K-major, 128-byte swizzle) into a 4-stage ring;
//   warp 1   owns the TMEM allocation (2 accumulators of BN fp32 columns);
//            one lane issues tcgen05.mma (M=128, N=BN, K=16, bf16 x bf16 ->
//            fp32) and tcgen05.commit to release ring stages and to publish
//            a finished accumulator;
//   warps 2-5 epilogue: tcgen05.ld 32 columns at a time from their TMEM
//            lane quarter, + bias, ReLU, round to bf16 into swizzled shared
//            staging boxes, TMA bulk stores to global;
//            double-buffered accumulators let tile i's epilogue overlap
//            tile i+1's MMAs.
// Every mbarrier wait is bounded (%globaltimer); on expiry the CTA raises an
// error flag (dgfx_dense_check), the roles leave their loops, outstanding
// copies and MMAs are drained with bounded waits and TMEM is freed.
// No TMA multicast, no clusters.
#include <algorithm>
#include <map>

#include "tensor_core.cuh"

namespace dgfx {
namespace {

constexpr int kBM = 128;
constexpr int kBK = 64;
constexpr int kStages = 4;
constexpr int kThreads = 192;

__device__ unsigned int g_dense_err;

template <int BN>
struct DenseSmem {
  static constexpr uint32_t kA = kBM * kBK * 2;  // 16 KB
  static constexpr uint32_t kB = BN * kBK * 2;   // up to 32 KB
  static constexpr uint32_t kStage = kA + kB;
  static constexpr uint32_t kTmemCols = BN * 2 <= 32 ? 32 : BN * 2;  // two accumulators
  // Output staging per epilogue warp: up to two 32-row x 64-column boxes
  // (4 KB each, 128-byte swizzle) handed to TMA stores.
  static constexpr uint32_t kBoxes = BN >= 128 ? 2 : 1;
  static constexpr uint32_t kOutWarp = kBoxes * 4096;
  static constexpr uint32_t kOut = 4 * kOutWarp;
  static constexpr size_t kBytes =
      static_cast<size_t>(kStages) * kStage + kOut + 1024 /* align */ + 256 /* barriers */;
};

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(x), "r"(y)
               : "memory");
}

template <int BN>
__global__ void __launch_bounds__(kThreads, 1)
    dense_concat_kernel(const __grid_constant__ CUtensorMap tm_x1, const __grid_constant__ CUtensorMap tm_x2,
                        const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_y, int64_t m,
                        int32_t n, int32_t kb1, int32_t kb_total, const float* __restrict__ bias, int32_t relu) {
  using L = DenseSmem<BN>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // 128-byte swizzled tiles need 1024-byte aligned shared addresses.
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* out_stage = smem + kStages * L::kStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(out_stage + L::kOut);
  // bars: full[kStages], empty[kStages], acc_full[2], acc_empty[2], drain
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + kStages);
  const uint32_t accf0 = smem_u32(bars + 2 * kStages), acce0 = smem_u32(bars + 2 * kStages + 2);
  const uint32_t drain = smem_u32(bars + 2 * kStages + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int64_t m_tiles = (m + kBM - 1) / kBM;
  const int32_t n_tiles = n / BN;
  const int64_t tiles = m_tiles * n_tiles;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(accf0 + 8 * b, 1);
      mbar_init(acce0 + 8 * b, 4);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(L::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      uint32_t issued = 0;  // stages with a load issued in the current ring pass
      bool ok = true;
      for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        const int32_t mb = static_cast<int32_t>(t / n_tiles), nb = static_cast<int32_t>(t % n_tiles);
        for (int32_t kb = 0; kb < kb_total; ++kb) {
          if (!mbar_wait(empty0 + 8 * s, ph ^ 1u, abort_flag, &g_dense_err)) {
            ok = false;
            break;
          }
          const uint32_t a_dst = smem_u32(smem + s * L::kStage);
          const uint32_t b_dst = a_dst + L::kA;
          mbar_arrive_expect_tx(full0 + 8 * s, L::kStage);
          if (kb < kb1) {
            tma_load_2d(a_dst, &tm_x1, full0 + 8 * s, kb * kBK, mb * kBM);
          } else {
            tma_load_2d(a_dst, &tm_x2, full0 + 8 * s, (kb - kb1) * kBK, mb * kBM);
          }
          tma_load_2d(b_dst, &tm_w, full0 + 8 * s, kb * kBK, nb * BN);
          issued |= 1u << s;
          if (++s == kStages) {
            s = 0;
            ph ^= 1u;
            issued = 0;
          }
        }
      }
      if (!ok) {
        // Drain: every stage loaded in this pass completes its transaction.
        for (int j = 0; j < kStages; ++j) {
          if (issued & (1u << j)) {
            const uint64_t t0 = now_ns();
            while (!mbar_test(full0 + 8 * j, ph) && now_ns() - t0 < kWaitNs) __nanosleep(100);
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_bf16(kBM, BN);
      int s = 0;
      uint32_t ph = 0;
      int b = 0;
      uint32_t aph = 0;
      bool ok = true;
      bool any = false;
      for (int64_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        if (!mbar_wait(acce0 + 8 * b, aph ^ 1u, abort_flag, &g_dense_err)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(b * BN);
        for (int32_t kb = 0; kb < kb_total; ++kb) {
          if (!mbar_wait(full0 + 8 * s, ph, abort_flag, &g_dense_err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + s * L::kStage);
          const uint64_t adesc = smem_desc_sw128(a_addr);
          const uint64_t bdesc = smem_desc_sw128(a_addr + L::kA);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) {
            // K step of 16 bf16 = 32 bytes inside the 128-byte swizzle atom.
            mma_bf16(d_tmem, adesc + 2 * k, bdesc + 2 * k, idesc, (kb | k) != 0 ? 1u : 0u);
          }
          any = true;
          mma_commit(empty0 + 8 * s);
          if (++s == kStages) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (!ok) break;
        mma_commit(accf0 + 8 * b);
        if (++b == 2) {
          b = 0;
          aph ^= 1u;
        }
      }
      if (any) {
        // All MMAs issued by this thread are complete once `drain` fires.
        mma_commit(drain);
        const uint64_t t0 = now_ns();
        while (!mbar_test(drain, 0) && now_ns() - t0 < kWaitNs) __nanosleep(100);
      }
    }
    __syncwarp();
  } else {
    // Epilogue: warp w reads TMEM lanes 32 * (w % 4) .. + 31 (its 32 rows),
    // 32 columns per tcgen05.ld; rounded bf16 rows go to this warp's staging
    // boxes in the 128-byte swizzled layout (16-byte chunk j of row r at
    // chunk j ^ (r % 8)) and leave in 32x64 TMA stores (rows past m are
    // clipped by the tensor map).
    const int q = warp & 3;
    const uint32_t lane_off = static_cast<uint32_t>(32 * q) << 16;
    uint8_t* my_stage = out_stage + (warp - 2) * L::kOutWarp;
    const uint32_t my_stage_u32 = smem_u32(my_stage);
    constexpr int kGroupCols = L::kBoxes * 64;
    int b = 0;
    uint32_t aph = 0;
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
      bool ready = true;
      if (lane == 0) ready = mbar_wait(accf0 + 8 * b, aph, abort_flag, &g_dense_err);
      ready = __shfl_sync(0xffffffffu, ready ? 1 : 0, 0) != 0;
      if (!ready) break;
      tc_fence_after();
      const int64_t mb = t / n_tiles;
      const int32_t nb = static_cast<int32_t>(t % n_tiles);
      const int64_t row0 = mb * kBM + 32 * q;
#pragma unroll 1
      for (int g = 0; g < BN / kGroupCols; ++g) {
        // The staging boxes are free once the previous stores read them.
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
#pragma unroll 1
        for (int cc = 0; cc < kGroupCols / 32; ++cc) {
          const int c = g * (kGroupCols / 32) + cc;
          uint32_t v[32];
          float bv[32];
          if (bias != nullptr) {
            const float4* b4 = reinterpret_cast<const float4*>(bias + nb * BN + c * 32);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 f = __ldg(b4 + j);
              bv[4 * j] = f.x;
              bv[4 * j + 1] = f.y;
              bv[4 * j + 2] = f.z;
              bv[4 * j + 3] = f.w;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) bv[j] = 0.0f;
          }
          tmem_ld32(tmem_base + lane_off + static_cast<uint32_t>(b * BN + c * 32), v);
          uint32_t packed[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float x0 = __uint_as_float(v[2 * j]) + bv[2 * j];
            float x1 = __uint_as_float(v[2 * j + 1]) + bv[2 * j + 1];
            if (relu) {
              x0 = fmaxf(x0, 0.0f);
              x1 = fmaxf(x1, 0.0f);
            }
            const __nv_bfloat162 h = __floats2bfloat162_rn(x0, x1);
            packed[j] = *reinterpret_cast<const uint32_t*>(&h);
          }
          uint8_t* box = my_stage + (cc >> 1) * 4096 + lane * 128;
          const int half = cc & 1;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int chunk = (half * 4 + j) ^ (lane & 7);
            *reinterpret_cast<uint4*>(box + chunk * 16) =
                make_uint4(packed[4 * j], packed[4 * j + 1], packed[4 * j + 2], packed[4 * j + 3]);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0 && row0 < m) {
#pragma unroll
          for (int bx = 0; bx < static_cast<int>(L::kBoxes); ++bx) {
            tma_store_2d(&tm_y, my_stage_u32 + bx * 4096, nb * BN + g * kGroupCols + bx * 64,
                         static_cast<int32_t>(row0));
          }
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acce0 + 8 * b);
      if (++b == 2) {
        b = 0;
        aph ^= 1u;
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(L::kTmemCols)
                 : "memory");
  }
}

template <int BN>
int launch_dense(const CUtensorMap& x1, const CUtensorMap& x2, const CUtensorMap& w, const CUtensorMap& ym, int64_t m,
                 int32_t n, int32_t kb1, int32_t kbt, const float* bias, int32_t relu, cudaStream_t stream) {
  using L = DenseSmem<BN>;
  static std::once_flag once[64];
  int dev = 0;
  DGFX_CUDA_TRY(cudaGetDevice(&dev));
  cudaError_t attr_err = cudaSuccess;
  std::call_once(once[dev & 63], [&]() {
    attr_err = cudaFuncSetAttribute(dense_concat_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(L::kBytes));
  });
  DGFX_CUDA_TRY(attr_err);
  int sms = 148;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t tiles = ((m + kBM - 1) / kBM) * (n / BN);
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(tiles, sms)));
  dense_concat_kernel<BN><<<grid, kThreads, L::kBytes, stream>>>(x1, x2, w, ym, m, n, kb1, kbt, bias, relu);
  DGFX_CUDA_TRY(cudaGetLastError());
  return DGFX_OK;
}

}  // namespace

unsigned int* dense_err_word() {
  static std::mutex mu;
  static std::map<int, unsigned int*> cache;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return nullptr;
  std::lock_guard<std::mutex> lock(mu);
  auto it = cache.find(dev);
  if (it != cache.end()) return it->second;
  void* p = nullptr;
  if (cudaGetSymbolAddress(&p, g_dense_err) != cudaSuccess) return nullptr;
  cache[dev] = static_cast<unsigned int*>(p);
  return static_cast<unsigned int*>(p);
}

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace dgfx

using namespace dgfx;

extern "C" int dgfx_dense_concat_bf16(const void* d_x1, int64_t k1, const void* d_x2, int64_t k2, int64_t m,
                                      const void* d_w, const float* d_bias, int64_t n, int32_t relu, void* d_y,
                                      dgfx_stream stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  if (m < 0 || k1 < kBK || k1 % kBK != 0 || k2 < 0 || k2 % kBK != 0 || n < 64 || n % 64 != 0 || d_x1 == nullptr ||
      d_w == nullptr || (k2 > 0 && d_x2 == nullptr) || (m > 0 && d_y == nullptr)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT,
                "dgfx_dense_concat_bf16: need k1 >= 64, k1 and k2 multiples of 64, n a multiple of 64, non-null "
                "operands");
  }
  if (!aligned16(d_x1) || !aligned16(d_w) || (d_x2 != nullptr && !aligned16(d_x2)) || !aligned16(d_y) ||
      (d_bias != nullptr && !aligned16(d_bias))) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_dense_concat_bf16: operands must be 16-byte aligned");
  }
  if (m >= (int64_t(1) << 31) || n > (int64_t(1) << 20) || (k1 + k2) / kBK > (1 << 20)) {
    return fail(DGFX_ERR_UNSUPPORTED, "dgfx_dense_concat_bf16: sizes out of range");
  }
  if (m == 0) return DGFX_OK;
  if (dense_err_word() == nullptr) return fail(DGFX_ERR_CUDA, "dgfx_dense: status word unavailable");
  const int bn = n % 256 == 0 ? 256 : (n % 128 == 0 ? 128 : 64);
  CUtensorMap x1, x2, w;
  DGFX_TRY(make_map(&x1, d_x1, m, k1, kBM));
  DGFX_TRY(make_map(&x2, k2 > 0 ? d_x2 : d_x1, m, k2 > 0 ? k2 : k1, kBM));
  DGFX_TRY(make_map(&w, d_w, n, k1 + k2, static_cast<uint32_t>(bn)));
  CUtensorMap ym;
  DGFX_TRY(make_map(&ym, d_y, m, n, 32));
  const int32_t kb1 = static_cast<int32_t>(k1 / kBK), kbt = static_cast<int32_t>((k1 + k2) / kBK);
  const int32_t n32 = static_cast<int32_t>(n);
  switch (bn) {
    case 256:
      return launch_dense<256>(x1, x2, w, ym, m, n32, kb1, kbt, d_bias, relu, stream);
    case 128:
      return launch_dense<128>(x1, x2, w, ym, m, n32, kb1, kbt, d_bias, relu, stream);
    default:
      return launch_dense<64>(x1, x2, w, ym, m, n32, kb1, kbt, d_bias, relu, stream);
  }
}

extern "C" int dgfx_dense_check(dgfx_stream stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  unsigned int* word = dense_err_word();
  if (word == nullptr) return fail(DGFX_ERR_CUDA, "dgfx_dense: status word unavailable");
  unsigned int v = 0;
  DGFX_CUDA_TRY(cudaMemcpyAsync(&v, word, sizeof(v), cudaMemcpyDeviceToHost, stream));
  DGFX_CUDA_TRY(cudaStreamSynchronize(stream));
  if (v != 0) {
    DGFX_CUDA_TRY(cudaMemsetAsync(word, 0, sizeof(v), stream));
    DGFX_CUDA_TRY(cudaStreamSynchronize(stream));
    return fail(DGFX_ERR_INTERNAL, "dgfx_dense: a pipeline wait timed out; the output is invalid");
  }
  return DGFX_OK;
}
