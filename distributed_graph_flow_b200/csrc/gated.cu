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
// accumulate in fp32. That rounding is as large as the results' own: dX and dW
// are off by 2.3e-3 (2-norm, relative) instead of the 1.7e-3 of a single
// rounding to bf16. Keeping D in two bf16 terms would double both products
// (880 of 2090 us at the sizes below).
//
// One kernel body, four kinds of tile (128 rows by up to 256 accumulator
// columns per CTA, K-blocks of 64):
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
// Tiles of 256 columns run on pairs of CTAs (cta_group::2, 256 rows per
// pair): each CTA loads its own A rows and half of B (for kForward one of
// them Wg, the other Wu), so a K-block brings 32 KB into an SM instead of
// 48, which with the operand reads is what its shared memory can carry at
// the full MMA rate. Smaller products use single CTAs and 128 or 64 columns,
// to spread over the SMs.
// Warps: 0 TMA producer, 1 TMEM owner and MMA issuer (the pair's leader
// issues), then the epilogue warps: four, two or one per TMEM lane quarter and group of columns.
// Two accumulators: the epilogue of a tile runs beside the products of the next. Every wait is
// bounded and latched in the status word of dgfx_dense_check; on expiry the roles leave,
// copies and MMAs are drained and TMEM is freed. No multicast loads.
//
// Bound by the tensor cores where there are many rows (K = 512: 4 M N K flop
// against 2 M (K + N) bytes), at small ones by the chain of one tile. Measured at
// 500,000 rows, K = 256 + 256, N = 512, silu: forward 380 us by itself (1.38
// PFLOP/s), 465 to 505 us in a loop (1.04 to 1.13), where power holds the clock down; training
// 2.1 to 2.25 ms in a loop, by the box. Its kernels by themselves, at the full clock, take
// 1.8 ms: forward 380, kGates 550 (2 GB of X,
// dh and D, for which HBM alone takes 310), kInput 412, kWeights 464, finish 5. Tiles of 128 x
// 256 on single CTAs took 423, 779, 438 and 519. One row: 7 us.
#include <algorithm>

#include "layer_math.cuh"
#include "tensor_core.cuh"

namespace dgfx {
namespace {

constexpr int kBM = 128;  // rows per CTA
constexpr int kBK = 64;

enum { kForward = 0, kGates = 1, kInput = 2, kWeights = 3 };
template <int KIND>
constexpr bool kFollows = KIND == kInput || KIND == kWeights;  // launched behind another kernel of its call

struct Maps {
  CUtensorMap a1, a2, b1, b2, b3, b4;
};

struct Args {
  int64_t m;
  int32_t n, k1, k2;
  int32_t kb1, kb_total;  // K-blocks of the first operand pair, of both
  int32_t n_tiles, units_per_n;
  int32_t cb1;        // kWeights: column blocks of X1
  int32_t kb_split;   // kWeights: K-blocks per split
  int32_t act;
  const float* b_gate;
  const float* b_up;
  const __nv_bfloat16* dh;
  __nv_bfloat16* out;    // h, D, or dX1
  __nv_bfloat16* out2;   // dX2
  float* partial;        // kGates: [4 slots, 2 N] bias sums; kWeights: [splits, 2 N, K]
  unsigned int* err;
};

// Per CTA. NACC accumulator columns; 256 of them on a pair of CTAs. RES: the
// weights of a CTA's column block stay in shared memory (up to kResident
// K-blocks), and only A rows come by the ring (forward 404 us without, 385 with,
// kGates 600 and 550, at the sizes above).
constexpr int kResident = 8;
template <int KIND, int NACC, bool RES>
struct Layout {
  static constexpr int kGroup = NACC == 256 ? 2 : 1;            // CTAs that share a tile
  static constexpr int kEpilogueWarps = NACC == 256 ? 16 : 8;
  static constexpr int kThreads = 64 + 32 * kEpilogueWarps;
  static constexpr uint32_t kA = kBM * kBK * 2;
  static constexpr uint32_t kB = NACC / kGroup * kBK * 2;
  static constexpr uint32_t kStage = RES ? kA : kA + kB;
  static constexpr uint32_t kHeld = RES ? kResident * kB : 0;
  static constexpr uint32_t kOutWarp = 2048;  // staging bytes per epilogue warp
  static constexpr int kStages = RES || NACC != 256 ? 4 : 6;
  static constexpr uint32_t kTmemCols = 2 * NACC;
  static constexpr size_t kBytes = static_cast<size_t>(kStages) * kStage + kHeld + kEpilogueWarps * kOutWarp +
                                   NACC * sizeof(float) /* biases */ + 1024 /* align */ + 256 /* barriers */;
  static_assert(kBytes <= 232448, "shared memory of a CTA");
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
__device__ __forceinline__ void gate_forward(float2 (&g)[8], const float2 (&u)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) g[j] = mul2(act2_f<ACT>(g[j]), u[j]);
}

template <int ACT>
__device__ __forceinline__ void gate_backward(float2 (&g)[8], float2 (&u)[8], const float2 (&d)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float2 v, s;
    act2_both_f<ACT>(g[j], &v, &s);
    g[j] = mul2(mul2(d[j], u[j]), s);
    u[j] = mul2(d[j], v);
  }
}

// Sums 32 values (16 pairs) over the 32 lanes: lane l returns the total of
// value l.
__device__ __forceinline__ float transpose_sum(float2 (&v)[16]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const bool upper = (lane & (2 * o)) != 0;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float2 send = upper ? v[i] : v[i + o], keep = upper ? v[i + o] : v[i];
      v[i] = add2(keep, make_float2(__shfl_xor_sync(0xffffffffu, send.x, 2 * o),
                                    __shfl_xor_sync(0xffffffffu, send.y, 2 * o)));
    }
  }
  const bool odd = (lane & 1) != 0;
  const float send = odd ? v[0].x : v[0].y, keep = odd ? v[0].y : v[0].x;
  return keep + __shfl_xor_sync(0xffffffffu, send, 1);
}

__device__ __forceinline__ uint4 pack8(const float2* f) {
  return make_uint4(pack_bf16(f[0].x, f[0].y), pack_bf16(f[1].x, f[1].y), pack_bf16(f[2].x, f[2].y),
                    pack_bf16(f[3].x, f[3].y));
}

// The tiles of one CTA or pair (`unit`). Kinds with a fixed column block per
// unit walk down the row blocks; kWeights has one tile and one range of K-blocks.
template <int KIND, int GROUP>
struct Walk {
  int32_t unit, rank, nb, m_tiles, step, mb;
  int32_t kb_begin, kb_end;
  __device__ Walk(const Args& p) {
    rank = GROUP == 2 ? static_cast<int32_t>(cluster_rank()) : 0;
    unit = static_cast<int32_t>(blockIdx.x) / GROUP;
    nb = unit % p.n_tiles;
    if (KIND == kWeights) {
      m_tiles = 1;
      step = 1;
      mb = 0;
      kb_begin = unit / p.n_tiles * p.kb_split;
      kb_end = min(kb_begin + p.kb_split, p.kb_total);
    } else {
      mb = unit / p.n_tiles;
      step = p.units_per_n;
      m_tiles = static_cast<int32_t>((p.m + kBM * GROUP - 1) / (kBM * GROUP));
      kb_begin = 0;
      kb_end = p.kb_total;
    }
  }
  // First row of this CTA in row block mb.
  __device__ int32_t row(int32_t mb_) const { return (mb_ * GROUP + rank) * kBM; }
};

// kWeights: output tile `t` -> its first row in [dWg; dWu], the operand and
// first column of X, and that column in K.
struct WeightTile {
  int32_t row0, col0, kcol0, kcols;
  bool second;
  __device__ WeightTile(const Args& p, int32_t t, int tile_rows, int nacc) {
    const int32_t row_blocks = (2 * p.n + tile_rows - 1) / tile_rows;
    const int32_t col_blocks = p.n_tiles / row_blocks;
    const int32_t rb = t / col_blocks, cb = t - rb * col_blocks;
    row0 = rb * tile_rows;
    second = cb >= p.cb1;
    col0 = (second ? cb - p.cb1 : cb) * nacc;
    kcol0 = (second ? p.k1 : 0) + col0;
    kcols = (second ? p.k2 : p.k1) - col0;
  }
};

template <int GROUP>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x, int32_t y) {
  if (GROUP == 2) tma_load_2d_pair(dst, map, bar, x, y);
  else tma_load_2d(dst, map, bar, x, y);
}

// Operand tiles of one K-block: A to a_dst, B to b_dst (either may be left out).
template <int KIND, int NACC, bool DO_A, bool DO_B, int G>
__device__ __forceinline__ void load_stage(const Maps& maps, const Args& p, const Walk<KIND, G>& w, int32_t mb, int32_t kb,
                                           uint32_t a_dst, uint32_t b_dst, uint32_t bar) {
  if (KIND == kForward || KIND == kGates) {
    constexpr int BN = NACC / 2;
    const bool first = kb < p.kb1;
    const int32_t x = (first ? kb : kb - p.kb1) * kBK;
    if (DO_A) load_box<G>(a_dst, first ? &maps.a1 : &maps.a2, bar, x, w.row(mb));
    if (DO_B) {
      const CUtensorMap* gate = first ? &maps.b1 : &maps.b2;
      const CUtensorMap* up = first ? &maps.b3 : &maps.b4;
      if (G == 2) {
        load_box<G>(b_dst, w.rank == 0 ? gate : up, bar, x, w.nb * BN);
      } else {
        load_box<G>(b_dst, gate, bar, x, w.nb * BN);
        load_box<G>(b_dst + BN * kBK * 2, up, bar, x, w.nb * BN);
      }
    }
  } else if (KIND == kInput) {
    const bool first = kb < p.kb1;
    const int32_t x = (first ? kb : kb - p.kb1) * kBK;
    load_box<G>(a_dst, first ? &maps.a1 : &maps.a2, bar, x, w.row(mb));
#pragma unroll
    for (int j = 0; j < NACC / G / 64; ++j) {
      load_box<G>(b_dst + j * 8192, first ? &maps.b1 : &maps.b2, bar, w.nb * NACC + w.rank * (NACC / G) + j * 64, x);
    }
  } else {
    const WeightTile t(p, w.nb, kBM * G, NACC);
#pragma unroll
    for (int j = 0; j < kBM / 64; ++j) {
      load_box<G>(a_dst + j * 8192, &maps.a1, bar, t.row0 + w.rank * kBM + j * 64, kb * kBK);
    }
#pragma unroll
    for (int j = 0; j < NACC / G / 64; ++j) {
      load_box<G>(b_dst + j * 8192, t.second ? &maps.b2 : &maps.b1, bar, t.col0 + w.rank * (NACC / G) + j * 64, kb * kBK);
    }
  }
}

// Writes a warp's staged 32 rows x P pieces of bf16 to rows row0.. of `out`
// ([m, pitch], this block of columns starting at col0, `limit` columns left).
template <int P>
__device__ __forceinline__ void store_bf16(const uint8_t* stage, __nv_bfloat16* out, int32_t pitch, int64_t row0,
                                           int64_t m, int32_t col0, int32_t limit) {
  const int lane = threadIdx.x & 31, r0 = lane / P, j = lane % P;
  __nv_bfloat16* to = out + row0 * pitch + col0 + r0 * pitch + j * 8;
  if (row0 + 32 <= m && P * 8 <= limit) {
#pragma unroll
    for (int k = 0; k < P; ++k) {
      *reinterpret_cast<uint4*>(to + k * (32 / P) * pitch) =
          *reinterpret_cast<const uint4*>(stage + piece_at<P>(r0 + k * (32 / P), j));
    }
  } else if (j * 8 < limit) {
#pragma unroll
    for (int k = 0; k < P; ++k) {
      if (row0 + r0 + k * (32 / P) < m) {
        *reinterpret_cast<uint4*>(to + k * (32 / P) * pitch) =
            *reinterpret_cast<const uint4*>(stage + piece_at<P>(r0 + k * (32 / P), j));
      }
    }
  }
}

// g and u of 16 columns from the accumulators, biases added (16-byte reads,
// the same for every lane).
__device__ __forceinline__ void load_gates(uint32_t acc_g, uint32_t acc_u, const float* bias_g, const float* bias_u,
                                           float2 (&g)[8], float2 (&u)[8]) {
  uint32_t gr[16], ur[16];
  tmem_ld_2x16(acc_g, acc_u, gr, ur);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float4 bg = reinterpret_cast<const float4*>(bias_g)[j], bu = reinterpret_cast<const float4*>(bias_u)[j];
    g[2 * j] = add2(make_float2(__uint_as_float(gr[4 * j]), __uint_as_float(gr[4 * j + 1])), make_float2(bg.x, bg.y));
    g[2 * j + 1] =
        add2(make_float2(__uint_as_float(gr[4 * j + 2]), __uint_as_float(gr[4 * j + 3])), make_float2(bg.z, bg.w));
    u[2 * j] = add2(make_float2(__uint_as_float(ur[4 * j]), __uint_as_float(ur[4 * j + 1])), make_float2(bu.x, bu.y));
    u[2 * j + 1] =
        add2(make_float2(__uint_as_float(ur[4 * j + 2]), __uint_as_float(ur[4 * j + 3])), make_float2(bu.z, bu.w));
  }
}

template <int KIND, int NACC, bool RES>
__device__ __forceinline__ void gated_body(const Maps& maps, const Args& p) {
  using L = Layout<KIND, NACC, RES>;
  constexpr int G = L::kGroup, BN = NACC / 2, S = L::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // 128-byte swizzled tiles need 1024-byte aligned shared addresses (the same
  // offset in both CTAs of a pair).
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* held = smem + S * L::kStage;
  uint8_t* out_stage = held + L::kHeld;
  float* biases = reinterpret_cast<float*>(out_stage + L::kEpilogueWarps * L::kOutWarp);
  uint64_t* bars = reinterpret_cast<uint64_t*>(biases + NACC);
  // bars: full[S], empty[S], acc_full[2], acc_empty[2], drain, held
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * S + 6);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + S);
  const uint32_t accf0 = smem_u32(bars + 2 * S), acce0 = smem_u32(bars + 2 * S + 2);
  const uint32_t drain = smem_u32(bars + 2 * S + 4), held_bar = smem_u32(bars + 2 * S + 5);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Walk<KIND, G> w(p);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(accf0 + 8 * b, 1);
      mbar_init(acce0 + 8 * b, G * L::kEpilogueWarps);
    }
    mbar_init(drain, 1);
    mbar_init(held_bar, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (KIND == kForward || KIND == kGates) {
    for (int i = threadIdx.x; i < NACC; i += L::kThreads) {
      const int32_t col = w.nb * BN + (i < BN ? i : i - BN);
      const float* b = i < BN ? p.b_gate : p.b_up;
      biases[i] = b != nullptr && col < p.n ? b[col] : 0.0f;
    }
  }
  if (warp == 1) {
    if (G == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(L::kTmemCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(L::kTmemCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  // Going backward the kernels form a chain: what is above runs beside the
  // end of the one before.
  let_next_start();
  if (kFollows<KIND>) after_previous();
  tc_fence_before();
  __syncthreads();
  if (G == 2) cluster_sync();  // the peer's barriers are ready
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      // Loads report to the leader's barriers.
      const uint32_t report0 = G == 2 ? map_rank(full0, 0) : full0;
      int s = 0;
      uint32_t ph = 0;
      uint32_t issued = 0;  // stages with a load issued in the current ring pass
      bool ok = true;
      if (RES) {  // the weights of this column block, once
        if (w.rank == 0) mbar_arrive_expect_tx(held_bar, G * L::kB * static_cast<uint32_t>(w.kb_end));
        const uint32_t report = G == 2 ? map_rank(held_bar, 0) : held_bar;
        for (int32_t kb = 0; kb < w.kb_end; ++kb) {
          load_stage<KIND, NACC, false, true, G>(maps, p, w, 0, kb, 0u, smem_u32(held + kb * L::kB), report);
        }
      }
      for (int32_t mb = w.mb; mb < w.m_tiles && ok; mb += w.step) {
        for (int32_t kb = w.kb_begin; kb < w.kb_end; ++kb) {
          if (!mbar_wait(empty0 + 8 * s, ph ^ 1u, abort_flag, p.err)) {
            ok = false;
            break;
          }
          if (w.rank == 0) mbar_arrive_expect_tx(full0 + 8 * s, G * L::kStage);
          const uint32_t a_dst = smem_u32(smem + s * L::kStage);
          load_stage<KIND, NACC, true, !RES, G>(maps, p, w, mb, kb, a_dst, a_dst + L::kA, report0 + 8 * s);
          issued |= 1u << s;
          if (++s == S) {
            s = 0;
            ph ^= 1u;
            issued = 0;
          }
        }
      }
      if (!ok) {
        // Drain: every stage loaded in this pass completes its transaction.
        // The second CTA of a pair cannot see it and gives its copies time.
        const uint64_t t1 = now_ns();
        while (w.rank != 0 && now_ns() - t1 < 10000000ull) __nanosleep(1000);
        for (int j = 0; j < S && w.rank == 0; ++j) {
          if (issued & (1u << j)) {
            const uint64_t t0 = now_ns();
            while (!mbar_test(full0 + 8 * j, ph) && now_ns() - t0 < kWaitNs) __nanosleep(100);
          }
        }
        if (RES && w.rank == 0) {
          const uint64_t t0 = now_ns();
          while (!mbar_test(held_bar, 0) && now_ns() - t0 < kWaitNs) __nanosleep(100);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && w.rank == 0) {
      constexpr bool kAMn = KIND == kWeights, kBMn = KIND == kWeights || KIND == kInput;
      constexpr uint32_t idesc = idesc_bf16(kBM * G, NACC, kAMn, kBMn);
      // A K step of 16: 32 bytes inside the swizzle atom, or 16 rows of 128.
      constexpr uint32_t kAStep = kAMn ? 2048 >> 4 : 32 >> 4, kBStep = kBMn ? 2048 >> 4 : 32 >> 4;
      auto commit = [](uint32_t bar) {
        if (G == 2) mma_commit_pair(bar);
        else mma_commit(bar);
      };
      int s = 0;
      uint32_t ph = 0;
      int b = 0;
      uint32_t aph = 0;
      bool ok = !RES || mbar_wait(held_bar, 0, abort_flag, p.err);
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
          const uint32_t b_addr = RES ? smem_u32(held) + static_cast<uint32_t>(kb) * L::kB : a_addr + L::kA;
          const uint64_t bdesc = kBMn ? smem_desc_sw128_mn(b_addr) : smem_desc_sw128(b_addr);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) {
            const uint32_t accumulate = (kb != w.kb_begin || k != 0) ? 1u : 0u;
            if (G == 2) mma_bf16_pair(d_tmem, adesc + kAStep * k, bdesc + kBStep * k, idesc, accumulate);
            else mma_bf16(d_tmem, adesc + kAStep * k, bdesc + kBStep * k, idesc, accumulate);
          }
          any = true;
          commit(empty0 + 8 * s);
          if (++s == S) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (!ok) break;
        commit(accf0 + 8 * b);
        if (++b == 2) {
          b = 0;
          aph ^= 1u;
        }
      }
      if (any) {
        // All MMAs issued by this thread are complete once `drain` fires.
        commit(drain);
        const uint64_t t0 = now_ns();
        while (!mbar_test(drain, 0) && now_ns() - t0 < kWaitNs) __nanosleep(100);
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3;            // TMEM lane quarter: rows 32 q ..
    const int part = (warp - 2) >> 2;  // this warp's group of columns
    constexpr int kParts = L::kEpilogueWarps / 4;
    const uint32_t lane_off = static_cast<uint32_t>(32 * q) << 16;
    uint8_t* stage = out_stage + (warp - 2) * L::kOutWarp;
    const uint32_t acce_leader = G == 2 ? map_rank(acce0, 0) : acce0;
    auto release = [&](int b) {  // this warp has read accumulator b
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (G == 2) mbar_arrive_cluster(acce_leader + 8 * b);
        else mbar_arrive(acce0 + 8 * b);
      }
    };
    int b = 0;
    uint32_t aph = 0;
    constexpr int GC = BN / kParts;  // columns of g and u per warp: 32, or 16 at 64 accumulator columns
    constexpr int kChunks = GC / 16;
    constexpr int GP = GC / 8;       // 16-byte pieces of them
    float bias_sum[kChunks];
    if (KIND == kGates) {
#pragma unroll
      for (int c = 0; c < kChunks; ++c) bias_sum[c] = 0.0f;
    }
    for (int32_t mb = w.mb; mb < w.m_tiles; mb += w.step) {
      const int64_t row0 = static_cast<int64_t>(w.row(mb)) + 32 * q;
      const bool row_ok = row0 + lane < p.m;
      const int32_t gcol0 = w.nb * BN + part * GC;
      // kGates: this warp's piece of dh, on its way while the products run.
      uint4 dh[GP];
      if (KIND == kGates) {
#pragma unroll
        for (int k = 0; k < GP; ++k) {
          const int i = lane + 32 * k, r = i / GP, j = i % GP;
          dh[k] = row0 + r < p.m && gcol0 + j * 8 < p.n
                      ? __ldg(reinterpret_cast<const uint4*>(p.dh + (row0 + r) * p.n + gcol0 + j * 8))
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
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int lc = part * GC + c * 16;
          float2 g[8], u[8];
          load_gates(acc + lc, acc + BN + lc, biases + lc, biases + BN + lc, g, u);
          switch (p.act) {
            case DGFX_ACT_RELU: gate_forward<DGFX_ACT_RELU>(g, u); break;
            case DGFX_ACT_SILU: gate_forward<DGFX_ACT_SILU>(g, u); break;
            case DGFX_ACT_GELU: gate_forward<DGFX_ACT_GELU>(g, u); break;
            case DGFX_ACT_SIGMOID: gate_forward<DGFX_ACT_SIGMOID>(g, u); break;
            default: gate_forward<DGFX_ACT_NONE>(g, u); break;
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            *reinterpret_cast<uint4*>(stage + piece_at<GP>(lane, c * 2 + j)) = pack8(g + 4 * j);
          }
        }
        release(b);
        store_bf16<GP>(stage, p.out, p.n, row0, p.m, gcol0, p.n - gcol0);
        __syncwarp();
      } else if (KIND == kGates) {
        uint4 du[GP];  // dg goes where dh was, du after it
#pragma unroll
        for (int k = 0; k < GP; ++k) {
          const int i = lane + 32 * k;
          *reinterpret_cast<uint4*>(stage + piece_at<GP>(i / GP, i % GP)) = dh[k];
        }
        __syncwarp();
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int lc = part * GC + c * 16;
          float2 g[8], u[8], d[8];
          load_gates(acc + lc, acc + BN + lc, biases + lc, biases + BN + lc, g, u);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float f[8];
            Vec16<__nv_bfloat16>::unpack(*reinterpret_cast<const uint4*>(stage + piece_at<GP>(lane, c * 2 + j)), f);
#pragma unroll
            for (int i = 0; i < 4; ++i) d[4 * j + i] = make_float2(f[2 * i], f[2 * i + 1]);
          }
          switch (p.act) {
            case DGFX_ACT_RELU: gate_backward<DGFX_ACT_RELU>(g, u, d); break;
            case DGFX_ACT_SILU: gate_backward<DGFX_ACT_SILU>(g, u, d); break;
            case DGFX_ACT_GELU: gate_backward<DGFX_ACT_GELU>(g, u, d); break;
            case DGFX_ACT_SIGMOID: gate_backward<DGFX_ACT_SIGMOID>(g, u, d); break;
            default: gate_backward<DGFX_ACT_NONE>(g, u, d); break;
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            *reinterpret_cast<uint4*>(stage + piece_at<GP>(lane, c * 2 + j)) = pack8(g + 4 * j);
            du[c * 2 + j] = pack8(u + 4 * j);
          }
          float2 v[16];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            v[j] = g[j];
            v[8 + j] = u[j];
          }
          if (row0 + 32 > p.m) {  // the last rows: nothing from behind the end
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = row_ok ? v[j] : make_float2(0.0f, 0.0f);
          }
          bias_sum[c] += transpose_sum(v);
        }
        release(b);
        store_bf16<GP>(stage, p.out, 2 * p.n, row0, p.m, gcol0, p.n - gcol0);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < GP; ++j) *reinterpret_cast<uint4*>(stage + piece_at<GP>(lane, j)) = du[j];
        __syncwarp();
        store_bf16<GP>(stage, p.out + p.n, 2 * p.n, row0, p.m, gcol0, p.n - gcol0);
        __syncwarp();
      } else if (KIND == kInput) {
        const int32_t kk = p.k1 + p.k2;
        constexpr int C = NACC / kParts;  // columns per warp, 32 staged at a time
#pragma unroll
        for (int cc = 0; cc < C / 32; ++cc) {
          const int lc = part * C + cc * 32;
          uint32_t v0[16], v1[16];
          tmem_ld_2x16(acc + lc, acc + lc + 16, v0, v1);
          if (cc + 1 == C / 32) release(b);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t o[4], o2[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              o[i] = pack_bf16(__uint_as_float(v0[8 * j + 2 * i]), __uint_as_float(v0[8 * j + 2 * i + 1]));
              o2[i] = pack_bf16(__uint_as_float(v1[8 * j + 2 * i]), __uint_as_float(v1[8 * j + 2 * i + 1]));
            }
            *reinterpret_cast<uint4*>(stage + piece_at<4>(lane, j)) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(stage + piece_at<4>(lane, 2 + j)) = make_uint4(o2[0], o2[1], o2[2], o2[3]);
          }
          __syncwarp();
          const int32_t col0 = w.nb * NACC + lc;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int i = lane + 32 * k, r = i / 4, j = i % 4;
            const int32_t col = col0 + j * 8;
            if (row0 + r < p.m && col < kk) {
              const uint4 v = *reinterpret_cast<const uint4*>(stage + piece_at<4>(r, j));
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
        const WeightTile t(p, w.nb, kBM * G, NACC);
        const int64_t kk = p.k1 + p.k2;
        float* out = p.partial + static_cast<int64_t>(w.unit / p.n_tiles) * 2 * p.n * kk;
        const int32_t n_row = t.row0 + w.rank * kBM + 32 * q;
        constexpr int C = NACC / kParts;  // columns per warp, 16 staged at a time
#pragma unroll 1
        for (int cc = 0; cc < C / 32; ++cc) {
          const int lc = part * C + cc * 32;
          uint32_t v[2][16];
          tmem_ld_2x16(acc + lc, acc + lc + 16, v[0], v[1]);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              *reinterpret_cast<uint4*>(stage + piece_at<4>(lane, j)) =
                  make_uint4(v[half][4 * j], v[half][4 * j + 1], v[half][4 * j + 2], v[half][4 * j + 3]);
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int i = lane + 32 * k, r = i / 4, j = i % 4;
              const int32_t col = lc + half * 16 + j * 4;
              if (n_row + r < 2 * p.n && col < t.kcols) {
                *reinterpret_cast<uint4*>(out + (n_row + r) * kk + t.kcol0 + col) =
                    *reinterpret_cast<const uint4*>(stage + piece_at<4>(r, j));
              }
            }
            __syncwarp();
          }
        }
        release(b);
      }
      if (++b == 2) {
        b = 0;
        aph ^= 1u;
      }
    }
    if (KIND == kGates) {
      // Lane l of a chunk holds the sum of column l of dg (l < 16) or du.
      const int64_t slot = (static_cast<int64_t>(w.unit / p.n_tiles) * G + w.rank) * 4 + q;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        const int32_t col = w.nb * BN + part * GC + c * 16 + (lane & 15);
        if (col < p.n) p.partial[(slot * 2 + (lane >> 4)) * p.n + col] = bias_sum[c];
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (G == 2) cluster_sync();  // the peer still reads this CTA's operands and barriers until here
  tc_fence_after();
  if (warp == 1) {
    if (G == 2) {
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(L::kTmemCols)
                   : "memory");
    } else {
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(L::kTmemCols)
                   : "memory");
    }
  }
}

template <int KIND, int NACC>
__global__ void __launch_bounds__(Layout<KIND, NACC, false>::kThreads, 1)
    gated_kernel(const __grid_constant__ Maps maps, const Args p) {
  gated_body<KIND, NACC, false>(maps, p);
}

template <int KIND, bool RES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Layout<KIND, 256, RES>::kThreads, 1)
    gated_pair_kernel(const __grid_constant__ Maps maps, const Args p) {
  gated_body<KIND, 256, RES>(maps, p);
}

// dW from the splits' fp32 tiles and the bias gradients from the CTAs' sums,
// both added in order (results do not change from run to run). The first
// `bias_blocks` blocks take 32 bias columns each (a warp adds every eighth
// slot, then the warps' sums are added), the others the weights.
__global__ void __launch_bounds__(256) gated_finish_kernel(const float* tiles, int32_t splits, int64_t n,
                                                           int64_t kk, uint2* __restrict__ dw_gate,
                                                           uint2* __restrict__ dw_up, const float* sums,
                                                           int32_t slots, int32_t bias_blocks,
                                                           float* __restrict__ db_gate, float* __restrict__ db_up) {
  __shared__ float part[8][32];
  after_previous();
  if (static_cast<int32_t>(blockIdx.x) < bias_blocks) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float s = 0.0f;
    if (i < 2 * n) {
#pragma unroll 8
      for (int32_t k = warp; k < slots; k += 8) s += sums[static_cast<int64_t>(k) * 2 * n + i];
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
      const float4 v = reinterpret_cast<const float4*>(tiles)[k * quads + i];
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

template <class K>
int launch(K kernel, bool follows, size_t smem, int threads, std::once_flag* once, const Maps& maps, const Args& p, int grid,
           cudaStream_t stream) {
  int dev = 0;
  DGFX_CUDA_TRY(cudaGetDevice(&dev));
  cudaError_t attr_err = cudaSuccess;
  std::call_once(once[dev & 63], [&]() {
    attr_err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  });
  DGFX_CUDA_TRY(attr_err);
  if (follows) launch_after(kernel, static_cast<unsigned>(grid), static_cast<unsigned>(threads), smem, stream, maps, p);
  else kernel<<<grid, threads, smem, stream>>>(maps, p);
  DGFX_CUDA_TRY(cudaGetLastError());
  return DGFX_OK;
}

template <int KIND, int NACC>
int launch_single(const Maps& maps, const Args& p, int units, cudaStream_t stream) {
  static std::once_flag once[64];
  using L = Layout<KIND, NACC, false>;
  return launch(gated_kernel<KIND, NACC>, kFollows<KIND>, L::kBytes, L::kThreads, once, maps, p, units, stream);
}

template <int KIND, bool RES>
int launch_pairs(const Maps& maps, const Args& p, int units, cudaStream_t stream) {
  static std::once_flag once[64];
  using L = Layout<KIND, 256, RES>;
  return launch(gated_pair_kernel<KIND, RES>, kFollows<KIND>, L::kBytes, L::kThreads, once, maps, p, 2 * units, stream);
}

// `units`: CTAs, or pairs of them at 256 accumulator columns.
template <int KIND>
int launch_nacc(int nacc, const Maps& maps, const Args& p, int units, cudaStream_t stream) {
  constexpr bool kHolds = KIND == kForward || KIND == kGates;
  if (nacc == 256) {
    if (kHolds && p.kb_total <= kResident) return launch_pairs<KIND, kHolds>(maps, p, units, stream);
    return launch_pairs<KIND, false>(maps, p, units, stream);
  }
  if (nacc == 128) return launch_single<KIND, 128>(maps, p, units, stream);
  return launch_single<KIND, 64>(maps, p, units, stream);
}

constexpr int kSms = 148;

// Accumulator columns: no wider than the product needs, and the widest tile
// that still gives every pair of CTAs, or half of the single ones, a tile: a narrow
// tile reads A more often but spreads a small product over the SMs (K = N = 256,
// 1000 rows: 4.9 us at 64 columns, 5.7 at 128, 8.2 on pairs; 20,000 rows: 17.9,
// 12.5 and 12.5; 32 outputs of 200,000 rows, K = 128: 13.4, 16.9 and 23.9). With
// fewer than half of the SMs at 128 columns, 64 columns take one wave too; above
// it they take two (4096 rows: 6.8 against 6.0 us).
int pick_nacc(int64_t m, int64_t cols) {
  if (cols <= 64) return 64;
  if (cols <= 128) return ceil_div(m, kBM) >= kSms ? 128 : 64;
  if (ceil_div(m, 2 * kBM) * ceil_div(cols, 256) >= kSms / 2) return 256;
  if (ceil_div(m, kBM) * ceil_div(cols, 128) >= kSms / 2) return 128;
  return 64;
}

struct Tiles {
  int nacc, n_tiles, units, units_per_n;  // units: CTAs or pairs; slots: CTAs that share a column block
  int slots() const { return units_per_n * (nacc == 256 ? 2 : 1); }
};

// A product with m rows and `cols` accumulator columns, column blocks fixed per unit.
Tiles plan_rows(int64_t m, int64_t cols) {
  Tiles t;
  t.nacc = pick_nacc(m, cols);
  const int group = t.nacc == 256 ? 2 : 1;
  t.n_tiles = static_cast<int>(ceil_div(cols, t.nacc));
  t.units_per_n = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>(ceil_div(m, kBM * group), kSms / group / t.n_tiles)));
  t.units = t.n_tiles * t.units_per_n;
  return t;
}

struct Plan {
  Tiles gate, input, weight;
  int splits, kb_split, cb1;
};

Plan make_plan(int64_t m, int64_t k1, int64_t k2, int64_t n) {
  Plan pl{};
  // Column blocks of the gate product hold half gate, half up columns.
  pl.gate = plan_rows(m, 2 * n);
  pl.input = plan_rows(m, k1 + k2);
  const int64_t widest = std::max(k1, k2), kb = std::max<int64_t>(ceil_div(m, kBK), 1);
  pl.weight.nacc = widest > 128 && 2 * n >= 256 ? 256 : (widest > 64 ? 128 : 64);
  const int group = pl.weight.nacc == 256 ? 2 : 1;
  pl.cb1 = static_cast<int>(ceil_div(k1, pl.weight.nacc));
  pl.weight.n_tiles = static_cast<int>(ceil_div(2 * n, kBM * group) * (pl.cb1 + ceil_div(k2, pl.weight.nacc)));
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(kb, kSms / group / pl.weight.n_tiles));
  pl.kb_split = static_cast<int>(ceil_div(kb, want));
  pl.splits = static_cast<int>(ceil_div(kb, pl.kb_split));
  pl.weight.units = pl.weight.n_tiles * pl.splits;
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
  w.sums = arena.take<float>(static_cast<size_t>(pl.gate.slots()) * 4 * 2 * n);
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
  DGFX_TRY(gate_maps(&maps, d_x1, k1, d_x2, k2, m, d_w_gate, d_w_up, n, pl.gate.nacc));
  Args p{};
  p.m = m;
  p.n = static_cast<int32_t>(n);
  p.k1 = static_cast<int32_t>(k1);
  p.k2 = static_cast<int32_t>(k2);
  p.kb1 = static_cast<int32_t>(ceil_div(k1, kBK));
  p.kb_total = p.kb1 + static_cast<int32_t>(ceil_div(k2, kBK));
  p.n_tiles = pl.gate.n_tiles;
  p.units_per_n = pl.gate.units_per_n;
  p.act = activation;
  p.b_gate = d_b_gate;
  p.b_up = d_b_up;
  p.out = static_cast<__nv_bfloat16*>(d_h);
  p.err = err;
  return launch_nacc<kForward>(pl.gate.nacc, maps, p, pl.gate.units, stream);
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
  if (!ptr_aligned16(d_workspace)) {
    return fail(DGFX_ERR_INVALID_ARGUMENT, std::string(who) + ": the workspace must be 16-byte aligned");
  }
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
    DGFX_TRY(gate_maps(&maps, d_x1, k1, d_x2, k2, m, d_w_gate, d_w_up, n, pl.gate.nacc));
    Args a = p;
    a.kb1 = static_cast<int32_t>(ceil_div(k1, kBK));
    a.kb_total = a.kb1 + static_cast<int32_t>(ceil_div(k2, kBK));
    a.n_tiles = pl.gate.n_tiles;
    a.units_per_n = pl.gate.units_per_n;
    a.act = activation;
    a.b_gate = d_b_gate;
    a.b_up = d_b_up;
    a.dh = static_cast<const __nv_bfloat16*>(d_dh);
    a.out = ws.d;
    a.partial = ws.sums;
    DGFX_TRY(launch_nacc<kGates>(pl.gate.nacc, maps, a, pl.gate.units, stream));
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
    a.n_tiles = pl.input.n_tiles;
    a.units_per_n = pl.input.units_per_n;
    a.out = static_cast<__nv_bfloat16*>(d_dx1);
    a.out2 = static_cast<__nv_bfloat16*>(d_dx2);
    DGFX_TRY(launch_nacc<kInput>(pl.input.nacc, maps, a, pl.input.units, stream));
  }
  if (d_dw_gate != nullptr) {
    Maps maps{};
    DGFX_TRY(make_map(&maps.a1, ws.d, m, 2 * n, kBK));
    DGFX_TRY(make_map(&maps.b1, d_x1, m, k1, kBK));
    DGFX_TRY(make_map(&maps.b2, k2 > 0 ? d_x2 : d_x1, m, k2 > 0 ? k2 : k1, kBK));
    Args a = p;
    a.kb_total = static_cast<int32_t>(ceil_div(m, kBK));
    a.kb_split = pl.kb_split;
    a.n_tiles = pl.weight.n_tiles;
    a.cb1 = pl.cb1;
    a.partial = ws.tiles;
    DGFX_TRY(launch_nacc<kWeights>(pl.weight.nacc, maps, a, pl.weight.units, stream));
  }
  if (d_dw_gate != nullptr || d_db_gate != nullptr || d_db_up != nullptr) {
    const int64_t bias_blocks = d_db_gate != nullptr || d_db_up != nullptr ? ceil_div(2 * n, 32) : 0;
    const int64_t weight_blocks = d_dw_gate != nullptr ? std::min<int64_t>(ceil_div(2 * n * kk / 4, 256), kSms * 8) : 0;
    launch_after(gated_finish_kernel, static_cast<unsigned>(bias_blocks + weight_blocks), 256, 0, stream, ws.tiles,
                 pl.splits, n, kk, static_cast<uint2*>(d_dw_gate), static_cast<uint2*>(d_dw_up), ws.sums,
                 pl.gate.slots() * 4, bias_blocks, d_db_gate, d_db_up);
    DGFX_CUDA_TRY(cudaGetLastError());
  }
  return DGFX_OK;
}
