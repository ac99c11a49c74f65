// Gated dense layer over a concat, forward and backward, on the
// 5th-generation tensor cores.
//
// With X = [X1 | X2] [M, K] (never materialised), Wg, Wu [N, K]:
//   g = X Wg^T + bg,  u = X Wu^T + bu,  h = act(g) * u.
// Backward from dh: g and u are computed again (4 M N K flop, instead of
// keeping 4 M N bytes of them rounded to bf16), then
//   du = dh act(g),  dg = dh u act'(g)     -> D = [dg | du], bf16 [M, 2 N]
//   dX = dg Wg + du Wu,  [dWg; dWu] = D^T X,  dbg, dbu = column sums.
// D is rounded once, to be a matrix operand of the two products that follow;
// the bias gradients are summed from its fp32 values before that. Products
// accumulate in fp32.
//
// One kernel body, four kinds of tile (128 rows by up to 256 accumulator
// columns, K-blocks of 64):
//   kForward  A = X (K-major), B = BN rows of Wg above BN rows of Wu: one MMA
//             gives the tile's g and u side by side in TMEM, and the
//             epilogue writes h; neither projection leaves the SM.
//   kGates    the same product; the epilogue reads dh and writes D, and
//             keeps the column sums of its CTA (every CTA has one column
//             block) in registers.
//   kInput    dX: A = D (K-major), B = W read MN-major (its rows are the
//             contraction): no transposed copy of the weights.
//   kWeights  dW: A = D, B = X, both MN-major (the contraction runs down the
//             rows of both); the rows are split over CTAs, whose fp32
//             tiles are added in order by gated_finish_kernel.
// Warps: 0 TMA producer, 1 TMEM owner and MMA issuer, 2-9 epilogue (two per
// TMEM lane quarter, half of the columns each). Two accumulators: the
// epilogue of a tile runs beside the products of the next. Every wait is
// bounded and latched in the status word of dgfx_dense_check; on expiry the roles leave,
// copies and MMAs are drained and TMEM is freed. No multicast, no clusters.
#include <algorithm>

#include "layer_math.cuh"
#include "tensor_core.cuh"

namespace dgfx {
namespace {

constexpr int kBM = 128;
constexpr int kBK = 64;
constexpr int kStages = 4;
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 64 + 32 * kEpilogueWarps;
constexpr uint32_t kStageOut = 4096;  // staging bytes per epilogue warp

enum { kForward = 0, kGates = 1, kInput = 2, kWeights = 3 };

struct Maps {
  CUtensorMap a1, a2, b1, b2, b3, b4;
};

struct Args {
  int64_t m;
  int32_t n, k1, k2;
  int32_t kb1, kb_total;  // K-blocks of the first operand pair, of both
  int32_t n_tiles, ctas_per_n;
  int32_t cb1;        // kWeights: column blocks of X1
  int32_t kb_split;   // kWeights: K-blocks per split
  int32_t act;
  const float* b_gate;
  const float* b_up;
  const __nv_bfloat16* dh;
  __nv_bfloat16* out;    // h, D, or dX1
  __nv_bfloat16* out2;   // dX2
  float* partial;        // kGates: [4 ctas_per_n, 2 N] bias sums; kWeights: [splits, 2 N, K]
  unsigned int* err;
};

template <int NACC>
struct Layout {
  static constexpr uint32_t kA = kBM * kBK * 2;
  static constexpr uint32_t kB = NACC * kBK * 2;
  static constexpr uint32_t kStage = kA + kB;
  static constexpr uint32_t kTmemCols = 2 * NACC;
  static constexpr size_t kBytes = static_cast<size_t>(kStages) * kStage + kEpilogueWarps * kStageOut +
                                   NACC * sizeof(float) /* biases */ + 1024 /* align */ + 256 /* barriers */;
};

// Two 16-column pieces of the accumulators (all 32 lanes of this warp's
// quarter), complete when it returns.
__device__ __forceinline__ void tmem_ld_2x16(uint32_t t0, uint32_t t1, uint32_t (&a)[16], uint32_t (&b)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%32];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%33];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]), "=r"(a[8]),
        "=r"(a[9]), "=r"(a[10]), "=r"(a[11]), "=r"(a[12]), "=r"(a[13]), "=r"(a[14]), "=r"(a[15]), "=r"(b[0]),
        "=r"(b[1]), "=r"(b[2]), "=r"(b[3]), "=r"(b[4]), "=r"(b[5]), "=r"(b[6]), "=r"(b[7]), "=r"(b[8]), "=r"(b[9]),
        "=r"(b[10]), "=r"(b[11]), "=r"(b[12]), "=r"(b[13]), "=r"(b[14]), "=r"(b[15])
      : "r"(t0), "r"(t1)
      : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Staging of 32 rows by P 16-byte pieces per warp: piece j of row r lies at
// piece j ^ f(r), so that both the row-wise writes (one row per lane) and the
// piece-wise reads (neighbouring lanes along a row) spread over the banks.
template <int P>
__device__ __forceinline__ uint32_t piece_at(int r, int j) {
  return static_cast<uint32_t>(r * P + (j ^ ((r / (8 / P)) & (P - 1)))) * 16u;
}

// act(g) * u, or the pair (dg, du), for 16 columns of one row.
template <int ACT>
__device__ __forceinline__ void gate_forward(float (&g)[16], const float (&u)[16]) {
#pragma unroll
  for (int j = 0; j < 16; ++j) g[j] = act_f<ACT>(g[j]) * u[j];
}

template <int ACT>
__device__ __forceinline__ void gate_backward(float (&g)[16], float (&u)[16], const float (&d)[16]) {
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    float v, s;
    act_both_f<ACT>(g[j], &v, &s);
    const float uj = u[j];
    u[j] = d[j] * v;
    g[j] = d[j] * uj * s;
  }
}

// Sums 32 values over the 32 lanes: lane l returns the total of v[l].
__device__ __forceinline__ float transpose_sum(float (&v)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool upper = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float send = upper ? v[i] : v[i + o];
      const float keep = upper ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0];
}

// The tiles of one CTA. Kinds with a fixed column block per CTA walk down the
// row blocks; kWeights has one tile and one range of K-blocks.
template <int KIND>
struct Walk {
  int32_t nb, m_tiles, step, mb;
  int32_t kb_begin, kb_end;
  __device__ Walk(const Args& p) {
    if (KIND == kWeights) {
      nb = static_cast<int32_t>(blockIdx.x) % p.n_tiles;  // output tile
      const int32_t split = static_cast<int32_t>(blockIdx.x) / p.n_tiles;
      m_tiles = 1;
      step = 1;
      mb = 0;
      kb_begin = split * p.kb_split;
      kb_end = min(kb_begin + p.kb_split, p.kb_total);
    } else {
      nb = static_cast<int32_t>(blockIdx.x) % p.n_tiles;
      mb = static_cast<int32_t>(blockIdx.x) / p.n_tiles;
      step = p.ctas_per_n;
      m_tiles = static_cast<int32_t>((p.m + kBM - 1) / kBM);
      kb_begin = 0;
      kb_end = p.kb_total;
    }
  }
};

// kWeights: output tile `t` -> half (0 gate, 1 up), its first row n0, the
// operand and first column of X, and that column in K.
struct WeightTile {
  int32_t half, n0, col0, kcol0, kcols;
  bool second;
  __device__ WeightTile(const Args& p, int32_t t, int nacc) {
    const int32_t row_blocks = (p.n + kBM - 1) / kBM;
    const int32_t col_blocks = p.n_tiles / (2 * row_blocks);
    const int32_t rb = t / col_blocks, cb = t - rb * col_blocks;
    half = rb / row_blocks;
    n0 = (rb - half * row_blocks) * kBM;
    second = cb >= p.cb1;
    col0 = (second ? cb - p.cb1 : cb) * nacc;
    kcol0 = (second ? p.k1 : 0) + col0;
    kcols = (second ? p.k2 : p.k1) - col0;
  }
};

template <int KIND, int NACC>
__device__ __forceinline__ void load_stage(const Maps& maps, const Args& p, const Walk<KIND>& w, int32_t mb, int32_t kb,
                                           uint32_t a_dst, uint32_t bar) {
  constexpr int BN = NACC / 2;
  const uint32_t b_dst = a_dst + Layout<NACC>::kA;
  if (KIND == kForward || KIND == kGates) {
    const bool first = kb < p.kb1;
    const int32_t x = (first ? kb : kb - p.kb1) * kBK;
    tma_load_2d(a_dst, first ? &maps.a1 : &maps.a2, bar, x, mb * kBM);
    tma_load_2d(b_dst, first ? &maps.b1 : &maps.b2, bar, x, w.nb * BN);
    tma_load_2d(b_dst + BN * kBK * 2, first ? &maps.b3 : &maps.b4, bar, x, w.nb * BN);
  } else if (KIND == kInput) {
    const bool first = kb < p.kb1;
    const int32_t x = (first ? kb : kb - p.kb1) * kBK;
    tma_load_2d(a_dst, first ? &maps.a1 : &maps.a2, bar, x, mb * kBM);
#pragma unroll
    for (int j = 0; j < NACC / 64; ++j) {
      tma_load_2d(b_dst + j * 8192, first ? &maps.b1 : &maps.b2, bar, w.nb * NACC + j * 64, x);
    }
  } else {
    const WeightTile t(p, w.nb, NACC);
#pragma unroll
    for (int j = 0; j < kBM / 64; ++j) {
      tma_load_2d(a_dst + j * 8192, &maps.a1, bar, t.half * p.n + t.n0 + j * 64, kb * kBK);
    }
#pragma unroll
    for (int j = 0; j < NACC / 64; ++j) {
      tma_load_2d(b_dst + j * 8192, t.second ? &maps.b2 : &maps.b1, bar, t.col0 + j * 64, kb * kBK);
    }
  }
}

// Writes a warp's staged 32 rows x P pieces of bf16 to rows row0.. of `out`
// ([m, pitch], this block of columns starting at col0, `limit` columns left).
template <int P>
__device__ __forceinline__ void store_bf16(const uint8_t* stage, __nv_bfloat16* out, int64_t pitch, int64_t row0,
                                           int64_t m, int32_t col0, int32_t limit) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k < P; ++k) {
    const int i = lane + 32 * k, r = i / P, j = i % P;
    if (row0 + r < m && j * 8 < limit) {
      *reinterpret_cast<uint4*>(out + (row0 + r) * pitch + col0 + j * 8) =
          *reinterpret_cast<const uint4*>(stage + piece_at<P>(r, j));
    }
  }
}

template <int KIND, int NACC>
__global__ void __launch_bounds__(kThreads, 1) gated_kernel(const __grid_constant__ Maps maps, const Args p) {
  using L = Layout<NACC>;
  constexpr int BN = NACC / 2;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // 128-byte swizzled tiles need 1024-byte aligned shared addresses.
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* out_stage = smem + kStages * L::kStage;
  float* biases = reinterpret_cast<float*>(out_stage + kEpilogueWarps * kStageOut);
  uint64_t* bars = reinterpret_cast<uint64_t*>(biases + NACC);
  // bars: full[kStages], empty[kStages], acc_full[2], acc_empty[2], drain
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 5);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + kStages);
  const uint32_t accf0 = smem_u32(bars + 2 * kStages), acce0 = smem_u32(bars + 2 * kStages + 2);
  const uint32_t drain = smem_u32(bars + 2 * kStages + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Walk<KIND> w(p);

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(accf0 + 8 * b, 1);
      mbar_init(acce0 + 8 * b, kEpilogueWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (KIND == kForward || KIND == kGates) {
    for (int i = threadIdx.x; i < NACC; i += kThreads) {
      const int32_t col = w.nb * BN + (i < BN ? i : i - BN);
      const float* b = i < BN ? p.b_gate : p.b_up;
      biases[i] = b != nullptr && col < p.n ? b[col] : 0.0f;
    }
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
      for (int32_t mb = w.mb; mb < w.m_tiles && ok; mb += w.step) {
        for (int32_t kb = w.kb_begin; kb < w.kb_end; ++kb) {
          if (!mbar_wait(empty0 + 8 * s, ph ^ 1u, abort_flag, p.err)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(full0 + 8 * s, L::kStage);
          load_stage<KIND, NACC>(maps, p, w, mb, kb, smem_u32(smem + s * L::kStage), full0 + 8 * s);
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
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr bool kAMn = KIND == kWeights, kBMn = KIND == kWeights || KIND == kInput;
      constexpr uint32_t idesc = idesc_bf16(kBM, NACC, kAMn, kBMn);
      // A K step of 16: 32 bytes inside the swizzle atom, or 16 rows of 128.
      constexpr uint32_t kAStep = kAMn ? 2048 >> 4 : 32 >> 4, kBStep = kBMn ? 2048 >> 4 : 32 >> 4;
      int s = 0;
      uint32_t ph = 0;
      int b = 0;
      uint32_t aph = 0;
      bool ok = true;
      bool any = false;
      for (int32_t mb = w.mb; mb < w.m_tiles && ok; mb += w.step) {
        if (!mbar_wait(acce0 + 8 * b, aph ^ 1u, abort_flag, p.err)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(b * NACC);
        for (int32_t kb = w.kb_begin; kb < w.kb_end; ++kb) {
          if (!mbar_wait(full0 + 8 * s, ph, abort_flag, p.err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + s * L::kStage);
          const uint64_t adesc = kAMn ? smem_desc_sw128_mn(a_addr) : smem_desc_sw128(a_addr);
          const uint64_t bdesc = kBMn ? smem_desc_sw128_mn(a_addr + L::kA) : smem_desc_sw128(a_addr + L::kA);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) {
            mma_bf16(d_tmem, adesc + kAStep * k, bdesc + kBStep * k, idesc, (kb != w.kb_begin || k != 0) ? 1u : 0u);
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
    const int q = warp & 3;             // TMEM lane quarter: rows 32 q ..
    const int half = (warp - 2) >> 2;   // half of the tile's columns
    const uint32_t lane_off = static_cast<uint32_t>(32 * q) << 16;
    uint8_t* stage = out_stage + (warp - 2) * kStageOut;
    int b = 0;
    uint32_t aph = 0;
    constexpr int kChunks = BN / 2 / 16;  // 16-column pieces of a warp's half (kForward, kGates)
    float bias_sum[kChunks];
    if (KIND == kGates) {
#pragma unroll
      for (int c = 0; c < kChunks; ++c) bias_sum[c] = 0.0f;
    }
    for (int32_t mb = w.mb; mb < w.m_tiles; mb += w.step) {
      const int64_t row0 = static_cast<int64_t>(mb) * kBM + 32 * q;
      const bool row_ok = row0 + lane < p.m;
      // kGates: the first piece of dh, on its way while the products run.
      constexpr int CW = BN / 2 < 32 ? BN / 2 : 32;  // columns staged at a time
      constexpr int GP = CW / 8;
      uint4 dh_next[GP];
      if (KIND == kGates) {
#pragma unroll
        for (int k = 0; k < GP; ++k) {
          const int i = lane + 32 * k, r = i / GP, j = i % GP;
          const int32_t col = w.nb * BN + half * (BN / 2) + j * 8;
          dh_next[k] = row0 + r < p.m && col < p.n
                           ? __ldg(reinterpret_cast<const uint4*>(p.dh + (row0 + r) * p.n + col))
                           : make_uint4(0, 0, 0, 0);
        }
      }
      bool ready = true;
      if (lane == 0) ready = mbar_wait(accf0 + 8 * b, aph, abort_flag, p.err);
      ready = __shfl_sync(0xffffffffu, ready ? 1 : 0, 0) != 0;
      if (!ready) break;
      tc_fence_after();
      const uint32_t acc = tmem_base + lane_off + static_cast<uint32_t>(b * NACC);

      if (KIND == kForward) {
        constexpr int P = BN / 16;  // 16-byte pieces per row of a warp's half
#pragma unroll 1
        for (int c = 0; c < kChunks; ++c) {
          const int lc = half * (BN / 2) + c * 16;
          uint32_t gr[16], ur[16];
          tmem_ld_2x16(acc + lc, acc + BN + lc, gr, ur);
          float g[16], u[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            g[j] = __uint_as_float(gr[j]) + biases[lc + j];
            u[j] = __uint_as_float(ur[j]) + biases[BN + lc + j];
          }
          switch (p.act) {
            case DGFX_ACT_RELU: gate_forward<DGFX_ACT_RELU>(g, u); break;
            case DGFX_ACT_SILU: gate_forward<DGFX_ACT_SILU>(g, u); break;
            case DGFX_ACT_GELU: gate_forward<DGFX_ACT_GELU>(g, u); break;
            case DGFX_ACT_SIGMOID: gate_forward<DGFX_ACT_SIGMOID>(g, u); break;
            default: gate_forward<DGFX_ACT_NONE>(g, u); break;
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            *reinterpret_cast<uint4*>(stage + piece_at<P>(lane, c * 2 + j)) =
                make_uint4(pack_bf16(g[8 * j], g[8 * j + 1]), pack_bf16(g[8 * j + 2], g[8 * j + 3]),
                           pack_bf16(g[8 * j + 4], g[8 * j + 5]), pack_bf16(g[8 * j + 6], g[8 * j + 7]));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acce0 + 8 * b);
        const int32_t col0 = w.nb * BN + half * (BN / 2);
        store_bf16<P>(stage, p.out, p.n, row0, p.m, col0, p.n - col0);
        __syncwarp();
      } else if (KIND == kGates) {
        uint8_t* stage2 = stage + kStageOut / 2;  // dg goes where dh was, du here
        constexpr int kSub = CW / 16;
#pragma unroll
        for (int cc = 0; cc < BN / 2 / CW; ++cc) {
#pragma unroll
          for (int k = 0; k < GP; ++k) {
            const int i = lane + 32 * k;
            *reinterpret_cast<uint4*>(stage + piece_at<GP>(i / GP, i % GP)) = dh_next[k];
          }
          if (cc + 1 < BN / 2 / CW) {
#pragma unroll
            for (int k = 0; k < GP; ++k) {
              const int i = lane + 32 * k, r = i / GP, j = i % GP;
              const int32_t col = w.nb * BN + half * (BN / 2) + (cc + 1) * CW + j * 8;
              dh_next[k] = row0 + r < p.m && col < p.n
                               ? __ldg(reinterpret_cast<const uint4*>(p.dh + (row0 + r) * p.n + col))
                               : make_uint4(0, 0, 0, 0);
            }
          }
          __syncwarp();
#pragma unroll
          for (int c = 0; c < kSub; ++c) {
            const int lc = half * (BN / 2) + cc * CW + c * 16;
            uint32_t gr[16], ur[16];
            tmem_ld_2x16(acc + lc, acc + BN + lc, gr, ur);
            float g[16], u[16], d[16];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float f[8];
              Vec16<__nv_bfloat16>::unpack(*reinterpret_cast<const uint4*>(stage + piece_at<GP>(lane, c * 2 + j)), f);
#pragma unroll
              for (int i = 0; i < 8; ++i) d[8 * j + i] = f[i];
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              g[j] = __uint_as_float(gr[j]) + biases[lc + j];
              u[j] = __uint_as_float(ur[j]) + biases[BN + lc + j];
            }
            switch (p.act) {
              case DGFX_ACT_RELU: gate_backward<DGFX_ACT_RELU>(g, u, d); break;
              case DGFX_ACT_SILU: gate_backward<DGFX_ACT_SILU>(g, u, d); break;
              case DGFX_ACT_GELU: gate_backward<DGFX_ACT_GELU>(g, u, d); break;
              case DGFX_ACT_SIGMOID: gate_backward<DGFX_ACT_SIGMOID>(g, u, d); break;
              default: gate_backward<DGFX_ACT_NONE>(g, u, d); break;
            }
            float v[32];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              v[j] = row_ok ? g[j] : 0.0f;
              v[16 + j] = row_ok ? u[j] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              *reinterpret_cast<uint4*>(stage + piece_at<GP>(lane, c * 2 + j)) =
                  make_uint4(pack_bf16(g[8 * j], g[8 * j + 1]), pack_bf16(g[8 * j + 2], g[8 * j + 3]),
                             pack_bf16(g[8 * j + 4], g[8 * j + 5]), pack_bf16(g[8 * j + 6], g[8 * j + 7]));
              *reinterpret_cast<uint4*>(stage2 + piece_at<GP>(lane, c * 2 + j)) =
                  make_uint4(pack_bf16(u[8 * j], u[8 * j + 1]), pack_bf16(u[8 * j + 2], u[8 * j + 3]),
                             pack_bf16(u[8 * j + 4], u[8 * j + 5]), pack_bf16(u[8 * j + 6], u[8 * j + 7]));
            }
            bias_sum[cc * kSub + c] += transpose_sum(v);
          }
          if (cc + 1 == BN / 2 / CW) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acce0 + 8 * b);
          } else {
            __syncwarp();
          }
          const int32_t col0 = w.nb * BN + half * (BN / 2) + cc * CW;
          store_bf16<GP>(stage, p.out, 2 * static_cast<int64_t>(p.n), row0, p.m, col0, p.n - col0);
          store_bf16<GP>(stage2, p.out + p.n, 2 * static_cast<int64_t>(p.n), row0, p.m, col0, p.n - col0);
          __syncwarp();
        }
      } else if (KIND == kInput) {
        const int32_t kk = p.k1 + p.k2;
#pragma unroll 1
        for (int cc = 0; cc < BN / 64 + (BN < 64 ? 1 : 0); ++cc) {
          constexpr int W = BN < 64 ? BN : 64;  // columns staged at a time
          constexpr int P = W / 8;
          const int lc = half * BN + cc * W;
#pragma unroll
          for (int c = 0; c < W / 32; ++c) {
            uint32_t v0[16], v1[16];
            tmem_ld_2x16(acc + lc + c * 32, acc + lc + c * 32 + 16, v0, v1);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t o[4], o2[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                o[i] = pack_bf16(__uint_as_float(v0[8 * j + 2 * i]), __uint_as_float(v0[8 * j + 2 * i + 1]));
                o2[i] = pack_bf16(__uint_as_float(v1[8 * j + 2 * i]), __uint_as_float(v1[8 * j + 2 * i + 1]));
              }
              *reinterpret_cast<uint4*>(stage + piece_at<P>(lane, c * 4 + j)) = make_uint4(o[0], o[1], o[2], o[3]);
              *reinterpret_cast<uint4*>(stage + piece_at<P>(lane, c * 4 + 2 + j)) =
                  make_uint4(o2[0], o2[1], o2[2], o2[3]);
            }
          }
          if (lc + W == (half + 1) * BN) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acce0 + 8 * b);
          } else {
            __syncwarp();
          }
          const int32_t col0 = w.nb * NACC + lc;
#pragma unroll
          for (int k = 0; k < P; ++k) {
            const int i = lane + 32 * k, r = i / P, j = i % P;
            const int32_t col = col0 + j * 8;
            if (row0 + r < p.m && col < kk) {
              const uint4 v = *reinterpret_cast<const uint4*>(stage + piece_at<P>(r, j));
              if (col < p.k1) {
                if (p.out != nullptr) *reinterpret_cast<uint4*>(p.out + (row0 + r) * p.k1 + col) = v;
              } else if (p.out2 != nullptr) {
                *reinterpret_cast<uint4*>(p.out2 + (row0 + r) * p.k2 + (col - p.k1)) = v;
              }
            }
          }
          __syncwarp();
        }
      } else {
        const WeightTile t(p, w.nb, NACC);
        const int64_t kk = p.k1 + p.k2;
        const int32_t split = static_cast<int32_t>(blockIdx.x) / p.n_tiles;
        float* out = p.partial + (static_cast<int64_t>(split) * 2 * p.n + static_cast<int64_t>(t.half) * p.n) * kk;
        const int32_t n_row = t.n0 + 32 * q;
#pragma unroll 1
        for (int cc = 0; cc < BN / 32; ++cc) {
          const int lc = half * BN + cc * 32;
          uint32_t v0[16], v1[16];
          tmem_ld_2x16(acc + lc, acc + lc + 16, v0, v1);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            *reinterpret_cast<uint4*>(stage + piece_at<8>(lane, j)) =
                make_uint4(v0[4 * j], v0[4 * j + 1], v0[4 * j + 2], v0[4 * j + 3]);
            *reinterpret_cast<uint4*>(stage + piece_at<8>(lane, 4 + j)) =
                make_uint4(v1[4 * j], v1[4 * j + 1], v1[4 * j + 2], v1[4 * j + 3]);
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int i = lane + 32 * k, r = i / 8, j = i % 8;
            if (n_row + r < p.n && lc + j * 4 < t.kcols) {
              *reinterpret_cast<uint4*>(out + (n_row + r) * kk + t.kcol0 + lc + j * 4) =
                  *reinterpret_cast<const uint4*>(stage + piece_at<8>(r, j));
            }
          }
          __syncwarp();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acce0 + 8 * b);
      }
      if (++b == 2) {
        b = 0;
        aph ^= 1u;
      }
    }
    if (KIND == kGates) {
      // Lane l of a piece holds the sum of column l of dg (l < 16) or du.
      const int64_t slot = (static_cast<int64_t>(blockIdx.x) / p.n_tiles) * 4 + q;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int32_t col = w.nb * BN + half * (BN / 2) + c * 16 + (lane & 15);
        if (col < p.n) p.partial[(slot * 2 + (lane >> 4)) * p.n + col] = bias_sum[c];
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(L::kTmemCols)
                 : "memory");
  }
}

// dW from the splits' fp32 tiles and the bias gradients from the CTAs' sums,
// both added in order (results do not change from run to run). The first
// `bias_blocks` blocks take 32 bias columns each (a warp adds every eighth
// slot, then the warps' sums are added), the others the weights.
__global__ void __launch_bounds__(256) gated_finish_kernel(const float* __restrict__ tiles, int32_t splits, int64_t n,
                                                           int64_t kk, uint2* __restrict__ dw_gate,
                                                           uint2* __restrict__ dw_up, const float* __restrict__ sums,
                                                           int32_t slots, int32_t bias_blocks,
                                                           float* __restrict__ db_gate, float* __restrict__ db_up) {
  __shared__ float part[8][32];
  if (static_cast<int32_t>(blockIdx.x) < bias_blocks) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float s = 0.0f;
    if (i < 2 * n) {
#pragma unroll 8
      for (int32_t k = warp; k < slots; k += 8) s += __ldg(sums + static_cast<int64_t>(k) * 2 * n + i);
    }
    part[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && i < 2 * n) {
      s = 0.0f;
      for (int k = 0; k < 8; ++k) s += part[k][lane];
      float* out = i < n ? db_gate : db_up;
      if (out != nullptr) out[i < n ? i : i - n] = s;
    }
    return;
  }
  const int64_t quads = 2 * n * kk / 4;
  const int64_t stride = static_cast<int64_t>(gridDim.x - bias_blocks) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x - bias_blocks) * blockDim.x + threadIdx.x; i < quads; i += stride) {
    float4 s = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int32_t k = 0; k < splits; ++k) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(tiles) + k * quads + i);
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
    const uint2 o = make_uint2(pack_bf16(s.x, s.y), pack_bf16(s.z, s.w));
    if (i < quads / 2) dw_gate[i] = o;
    else dw_up[i - quads / 2] = o;
  }
}

template <int KIND, int NACC>
int launch(const Maps& maps, const Args& p, int grid, cudaStream_t stream) {
  static std::once_flag once[64];
  int dev = 0;
  DGFX_CUDA_TRY(cudaGetDevice(&dev));
  cudaError_t attr_err = cudaSuccess;
  std::call_once(once[dev & 63], [&]() {
    attr_err = cudaFuncSetAttribute(gated_kernel<KIND, NACC>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(Layout<NACC>::kBytes));
  });
  DGFX_CUDA_TRY(attr_err);
  gated_kernel<KIND, NACC><<<grid, kThreads, Layout<NACC>::kBytes, stream>>>(maps, p);
  DGFX_CUDA_TRY(cudaGetLastError());
  return DGFX_OK;
}

template <int KIND>
int launch_nacc(int nacc, const Maps& maps, const Args& p, int grid, cudaStream_t stream) {
  switch (nacc) {
    case 256: return launch<KIND, 256>(maps, p, grid, stream);
    case 128: return launch<KIND, 128>(maps, p, grid, stream);
    default: return launch<KIND, 64>(maps, p, grid, stream);
  }
}

constexpr int kSms = 148;

// Accumulator columns: the widest tile that still gives every SM one (a
// narrow tile reads A more often but spreads a small product over the SMs).
int pick_nacc(int64_t m_tiles, int64_t cols, int per_col) {
  for (int nacc = 256; nacc > 64; nacc /= 2) {
    if (m_tiles * ceil_div(cols * per_col, nacc) >= kSms) return nacc;
  }
  return 64;
}

struct Plan {
  int64_t m_tiles;
  int nacc_gate, tiles_gate, ctas_gate;      // kForward, kGates
  int nacc_input, tiles_input, ctas_input;   // kInput
  int nacc_weight, tiles_weight, splits, kb_split, cb1;
};

Plan make_plan(int64_t m, int64_t k1, int64_t k2, int64_t n) {
  Plan pl{};
  pl.m_tiles = ceil_div(m, kBM);
  pl.nacc_gate = pick_nacc(pl.m_tiles, n, 2);
  pl.tiles_gate = static_cast<int>(ceil_div(2 * n, pl.nacc_gate));
  pl.ctas_gate = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(pl.m_tiles, kSms / pl.tiles_gate)));
  pl.nacc_input = pick_nacc(pl.m_tiles, k1 + k2, 1);
  pl.tiles_input = static_cast<int>(ceil_div(k1 + k2, pl.nacc_input));
  pl.ctas_input = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(pl.m_tiles, kSms / pl.tiles_input)));
  const int64_t row_blocks = 2 * ceil_div(n, kBM), kb = ceil_div(m, kBK);
  pl.nacc_weight = std::max(k1, k2) > 128 ? 256 : (std::max(k1, k2) > 64 ? 128 : 64);
  pl.cb1 = static_cast<int>(ceil_div(k1, pl.nacc_weight));
  pl.tiles_weight = static_cast<int>(row_blocks * (pl.cb1 + ceil_div(k2, pl.nacc_weight)));
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(kb, kSms / pl.tiles_weight));
  pl.kb_split = static_cast<int>(ceil_div(std::max<int64_t>(kb, 1), want));
  pl.splits = static_cast<int>(ceil_div(std::max<int64_t>(kb, 1), pl.kb_split));
  return pl;
}

struct Work {
  __nv_bfloat16* d;
  float *tiles, *sums;
  bool ok;
  size_t bytes;
};

Work carve(void* base, size_t cap, const Plan& pl, int64_t m, int64_t kk, int64_t n) {
  Arena arena(base, cap);
  Work w;
  w.d = arena.take<__nv_bfloat16>(static_cast<size_t>(m) * 2 * n);
  w.tiles = arena.take<float>(static_cast<size_t>(pl.splits) * 2 * n * kk);
  w.sums = arena.take<float>(static_cast<size_t>(pl.ctas_gate) * 4 * 2 * n);
  w.ok = arena.ok();
  w.bytes = arena.used;
  return w;
}

int check_shape(const char* who, int64_t m, int64_t k1, int64_t k2, int64_t n, int32_t act) {
  if (m < 0 || k1 < 8 || k1 % 8 != 0 || k2 < 0 || k2 % 8 != 0 || n < 8 || n % 8 != 0 || act < DGFX_ACT_NONE ||
      act > DGFX_ACT_SIGMOID) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, std::string(who) +
                                               ": need k1 >= 8, k1, k2 and n multiples of 8, a known activation");
  }
  if (m >= (int64_t(1) << 31) - kBM || n > (int64_t(1) << 20) || k1 + k2 > (int64_t(1) << 20)) {
    return fail(DGFX_ERR_UNSUPPORTED, std::string(who) + ": sizes out of range");
  }
  return DGFX_OK;
}

int gate_maps(Maps* maps, const void* x1, int64_t k1, const void* x2, int64_t k2, int64_t m, const void* wg,
              const void* wu, int64_t n, int nacc) {
  const int64_t kk = k1 + k2;
  const uint32_t bn = static_cast<uint32_t>(nacc / 2);
  const auto* g = static_cast<const __nv_bfloat16*>(wg);
  const auto* u = static_cast<const __nv_bfloat16*>(wu);
  DGFX_TRY(make_map(&maps->a1, x1, m, k1, kBM));
  DGFX_TRY(make_map(&maps->b1, g, n, k1, bn, kk));
  DGFX_TRY(make_map(&maps->b3, u, n, k1, bn, kk));
  // Without a second operand its maps are never used.
  DGFX_TRY(make_map(&maps->a2, k2 > 0 ? x2 : x1, m, k2 > 0 ? k2 : k1, kBM));
  DGFX_TRY(make_map(&maps->b2, k2 > 0 ? g + k1 : g, n, k2 > 0 ? k2 : k1, bn, kk));
  DGFX_TRY(make_map(&maps->b4, k2 > 0 ? u + k1 : u, n, k2 > 0 ? k2 : k1, bn, kk));
  return DGFX_OK;
}

}  // namespace
}  // namespace dgfx

using namespace dgfx;

extern "C" int dgfx_gated_dense_concat_bf16(const void* d_x1, int64_t k1, const void* d_x2, int64_t k2, int64_t m,
                                            const void* d_w_gate, const void* d_w_up, const float* d_b_gate,
                                            const float* d_b_up, int64_t n, int32_t activation, void* d_h,
                                            dgfx_stream stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  DGFX_TRY(check_shape("dgfx_gated_dense_concat_bf16", m, k1, k2, n, activation));
  if (m == 0) return DGFX_OK;
  if (d_x1 == nullptr || (k2 > 0 && d_x2 == nullptr) || d_w_gate == nullptr || d_w_up == nullptr || d_h == nullptr) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_dense_concat_bf16: null operand");
  }
  if (!ptr_aligned16(d_x1) || !ptr_aligned16(d_x2) || !ptr_aligned16(d_w_gate) || !ptr_aligned16(d_w_up) ||
      !ptr_aligned16(d_h)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_dense_concat_bf16: operands must be 16-byte aligned");
  }
  unsigned int* err = dense_err_word();
  if (err == nullptr) return fail(DGFX_ERR_CUDA, "dgfx_gated_dense_concat_bf16: status word unavailable");
  const Plan pl = make_plan(m, k1, k2, n);
  Maps maps{};
  DGFX_TRY(gate_maps(&maps, d_x1, k1, d_x2, k2, m, d_w_gate, d_w_up, n, pl.nacc_gate));
  Args p{};
  p.m = m;
  p.n = static_cast<int32_t>(n);
  p.k1 = static_cast<int32_t>(k1);
  p.k2 = static_cast<int32_t>(k2);
  p.kb1 = static_cast<int32_t>(ceil_div(k1, kBK));
  p.kb_total = p.kb1 + static_cast<int32_t>(ceil_div(k2, kBK));
  p.n_tiles = pl.tiles_gate;
  p.ctas_per_n = pl.ctas_gate;
  p.act = activation;
  p.b_gate = d_b_gate;
  p.b_up = d_b_up;
  p.out = static_cast<__nv_bfloat16*>(d_h);
  p.err = err;
  return launch_nacc<kForward>(pl.nacc_gate, maps, p, pl.tiles_gate * pl.ctas_gate, stream);
}

extern "C" int dgfx_gated_dense_concat_backward_workspace_size(int64_t k1, int64_t k2, int64_t m, int64_t n,
                                                               size_t* bytes) {
  DGFX_TRY(check_shape("dgfx_gated_dense_concat_backward_workspace_size", m, k1, k2, n, DGFX_ACT_NONE));
  if (bytes == nullptr) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, "dgfx_gated_dense_concat_backward_workspace_size: null result");
  }
  *bytes = carve(nullptr, 0, make_plan(m, k1, k2, n), m, k1 + k2, n).bytes;
  return DGFX_OK;
}

extern "C" int dgfx_gated_dense_concat_backward_bf16(const void* d_dh, const void* d_x1, int64_t k1, const void* d_x2,
                                                     int64_t k2, int64_t m, const void* d_w_gate, const void* d_w_up,
                                                     const float* d_b_gate, const float* d_b_up, int64_t n,
                                                     int32_t activation, void* d_dx1, void* d_dx2, void* d_dw_gate,
                                                     void* d_dw_up, float* d_db_gate, float* d_db_up,
                                                     void* d_workspace, size_t workspace_bytes, dgfx_stream stream_) {
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  const char* who = "dgfx_gated_dense_concat_backward_bf16";
  DGFX_TRY(check_shape(who, m, k1, k2, n, activation));
  if ((d_dw_gate == nullptr) != (d_dw_up == nullptr) || d_w_gate == nullptr || d_w_up == nullptr ||
      (m > 0 && (d_dh == nullptr || d_x1 == nullptr || (k2 > 0 && d_x2 == nullptr)))) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, std::string(who) + ": null operand (both weight gradients or neither)");
  }
  for (const void* q : {d_dh, d_x1, d_x2, d_w_gate, d_w_up, static_cast<const void*>(d_dx1),
                        static_cast<const void*>(d_dx2), static_cast<const void*>(d_dw_gate),
                        static_cast<const void*>(d_dw_up)}) {
    if (!ptr_aligned16(q)) return fail(DGFX_ERR_INVALID_ARGUMENT, std::string(who) + ": operands must be 16-byte aligned");
  }
  const int64_t kk = k1 + k2;
  if (m == 0) {
    if (d_dw_gate != nullptr) {
      DGFX_CUDA_TRY(cudaMemsetAsync(d_dw_gate, 0, 2 * n * kk, stream));
      DGFX_CUDA_TRY(cudaMemsetAsync(d_dw_up, 0, 2 * n * kk, stream));
    }
    if (d_db_gate != nullptr) DGFX_CUDA_TRY(cudaMemsetAsync(d_db_gate, 0, 4 * n, stream));
    if (d_db_up != nullptr) DGFX_CUDA_TRY(cudaMemsetAsync(d_db_up, 0, 4 * n, stream));
    return DGFX_OK;
  }
  const Plan pl = make_plan(m, k1, k2, n);
  const Work ws = carve(d_workspace, workspace_bytes, pl, m, kk, n);
  if (d_workspace == nullptr || !ws.ok) return fail(DGFX_ERR_WORKSPACE, std::string(who) + ": workspace too small");
  unsigned int* err = dense_err_word();
  if (err == nullptr) return fail(DGFX_ERR_CUDA, std::string(who) + ": status word unavailable");

  Args p{};
  p.m = m;
  p.n = static_cast<int32_t>(n);
  p.k1 = static_cast<int32_t>(k1);
  p.k2 = static_cast<int32_t>(k2);
  p.err = err;
  {  // D = [dg | du] and the bias sums
    Maps maps{};
    DGFX_TRY(gate_maps(&maps, d_x1, k1, d_x2, k2, m, d_w_gate, d_w_up, n, pl.nacc_gate));
    Args a = p;
    a.kb1 = static_cast<int32_t>(ceil_div(k1, kBK));
    a.kb_total = a.kb1 + static_cast<int32_t>(ceil_div(k2, kBK));
    a.n_tiles = pl.tiles_gate;
    a.ctas_per_n = pl.ctas_gate;
    a.act = activation;
    a.b_gate = d_b_gate;
    a.b_up = d_b_up;
    a.dh = static_cast<const __nv_bfloat16*>(d_dh);
    a.out = ws.d;
    a.partial = ws.sums;
    DGFX_TRY(launch_nacc<kGates>(pl.nacc_gate, maps, a, pl.tiles_gate * pl.ctas_gate, stream));
  }
  if (d_dx1 != nullptr || d_dx2 != nullptr) {
    Maps maps{};
    DGFX_TRY(make_map(&maps.a1, ws.d, m, n, kBM, 2 * n));
    DGFX_TRY(make_map(&maps.a2, ws.d + n, m, n, kBM, 2 * n));
    DGFX_TRY(make_map(&maps.b1, d_w_gate, n, kk, kBK));
    DGFX_TRY(make_map(&maps.b2, d_w_up, n, kk, kBK));
    Args a = p;
    a.kb1 = static_cast<int32_t>(ceil_div(n, kBK));
    a.kb_total = 2 * a.kb1;
    a.n_tiles = pl.tiles_input;
    a.ctas_per_n = pl.ctas_input;
    a.out = static_cast<__nv_bfloat16*>(d_dx1);
    a.out2 = static_cast<__nv_bfloat16*>(d_dx2);
    DGFX_TRY(launch_nacc<kInput>(pl.nacc_input, maps, a, pl.tiles_input * pl.ctas_input, stream));
  }
  if (d_dw_gate != nullptr) {
    Maps maps{};
    DGFX_TRY(make_map(&maps.a1, ws.d, m, 2 * n, kBK));
    DGFX_TRY(make_map(&maps.b1, d_x1, m, k1, kBK));
    DGFX_TRY(make_map(&maps.b2, k2 > 0 ? d_x2 : d_x1, m, k2 > 0 ? k2 : k1, kBK));
    Args a = p;
    a.kb_total = static_cast<int32_t>(ceil_div(m, kBK));
    a.kb_split = pl.kb_split;
    a.n_tiles = pl.tiles_weight;
    a.cb1 = pl.cb1;
    a.partial = ws.tiles;
    DGFX_TRY(launch_nacc<kWeights>(pl.nacc_weight, maps, a, pl.tiles_weight * pl.splits, stream));
  }
  if (d_dw_gate != nullptr || d_db_gate != nullptr || d_db_up != nullptr) {
    const int64_t bias_blocks = d_db_gate != nullptr || d_db_up != nullptr ? ceil_div(2 * n, 32) : 0;
    const int64_t weight_blocks = d_dw_gate != nullptr ? std::min<int64_t>(ceil_div(2 * n * kk / 4, 256), kSms * 8) : 0;
    gated_finish_kernel<<<static_cast<unsigned>(bias_blocks + weight_blocks), 256, 0, stream>>>(
        ws.tiles, pl.splits, n, kk, static_cast<uint2*>(d_dw_gate), static_cast<uint2*>(d_dw_up), ws.sums,
        pl.ctas_gate * 4, static_cast<int32_t>(bias_blocks), d_db_gate, d_db_up);
    DGFX_CUDA_TRY(cudaGetLastError());
  }
  return DGFX_OK;
}
