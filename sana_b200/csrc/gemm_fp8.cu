// 8-bit projection with one power-of-two scale for each block of 128 along K:
//
//   out[m][n] = epilogue( sum_kb 2^(ea[m][kb] + ew[n][kb]) * sum_{k in block kb} a[m][k] w[n][k] )
//
// a, w are E4M3 codes (K-major), ea / ew the exponents, stored as E8M0 bytes (exponent + 127) in a plain row-major
// matrix [ceil(rows / block_rows), blocks], block_rows 1 (activations) or 128 (weights).  A power of two costs the
// quantiser no rounding of its own (x * 2^-e is exact) and is what the tensor core applies itself
// (tcgen05.mma kind::mxf8f6f4 takes one E8M0 scale for each row and 32 K elements): the partial sums of a block never
// leave tensor memory, where a general fp32 scale would have to read them back after every 128 elements.
//
// The tensor core reads scales from tensor memory, as 4-column tiles of 128 rows x 4 bytes (byte b = scale b of the
// row; the instruction names the byte), filled from 512-byte shared-memory tiles [row % 32][row / 32][b].  One byte
// serves a whole stage here (K = 128 = four instructions), so a tile feeds four stages.  A warp of its own builds the
// tiles from the plain scale matrix - one 32-bit load per row gives the bytes of four stages - and copies them with
// tcgen05.cp, one tile ahead of the MMAs: weights are read in the layout they are stored in, nothing is repacked.
//
// Measured: 3.03 PFLOP/s at M = N = K = 8192 (bound by the tensor pipe).  4096 x 2240 -> 11200 with
// bias and SiLU 94 us, 16384 x 5600 -> 2240 with gate and residual 154 us (2.2 and 2.7 PFLOP/s: fewer K blocks per
// tile to hide an epilogue behind, and a last wave that is not full).  600 x 2304 -> 2240 10 us: 90 tiles, one each
// for 90 SMs, so the latency of one tile's pipeline and epilogue.
#include <cuda_fp8.h>

#include "tc_common.cuh"

namespace sana {

__device__ int g_fp8_status = 0;

constexpr int F8_BK = 128;                       // elements (= bytes) of a stage: one scale block, one swizzle row
constexpr int F8_GROUP = 4;                      // stages served by one scale tile
constexpr int F8_EPI_WARPS = 8;
constexpr int F8_THREADS = 128 + 32 * F8_EPI_WARPS;  // warp 0 loads, 1 MMA, 2 scales, 3 idle; then the epilogue warps
constexpr int F8_CTRL_BYTES = 256;
// block-scaled instruction descriptor: A = B = E4M3 (code 0), both K-major, scale type UE8M0 (bit 23), N>>3 at 17,
// M>>4 at 24; bits 4-5 / 29-30 name the byte of W's / A's scale word
constexpr uint32_t f8_idesc(int M, int N) { return (1u << 23) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }
__device__ __forceinline__ uint32_t f8_scale_byte(uint32_t b) { return (b << 4) | (b << 29); }

__device__ __forceinline__ void umma_fp8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                         uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
      : "memory");
}
__device__ __forceinline__ void umma_fp8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                              uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
      : "memory");
}

// Plain scale matrix of an operand: byte (row >> shift) * ld + block; ld and the base are multiples of 4 and every
// row can be read up to the next multiple of 4 blocks.
struct F8Scales {
  const unsigned char* p;
  int64_t ld;
  int64_t rows;  // operand rows
  int shift;     // 0: a scale per row, 7: per 128 rows
};
// this lane's 16 bytes of the tile of rows r0 .. r0 + 127, blocks 4 g .. 4 g + 3
__device__ __forceinline__ uint4 f8_scale_words(const F8Scales& s, int r0, int g, int lane) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = (int64_t)r0 + lane + 32 * i;
    w[i] = r < s.rows ? __ldg(reinterpret_cast<const uint32_t*>(s.p + (r >> s.shift) * s.ld + 4 * g)) : 0x7f7f7f7fu;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Bounded wait like mbar_wait, with the plain poll: the suspend hint may keep a warp asleep for up to a microsecond past the
// arrival, and the one accumulator passes from the products to the epilogue and back once a tile.
__device__ __forceinline__ bool f8_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
  if (mbar_try_wait_poll(bar, parity)) return true;
  const long long t0 = clock64();
  uint32_t spins = 0;
  while (!mbar_try_wait_poll(bar, parity)) {
    if ((++spins & 255u) == 0) {
      if (*abort_flag) return false;
      if (clock64() - t0 > TC_WAIT_LIMIT_CYCLES) {
        *abort_flag = code;
        atomicExch(&g_fp8_status, code);
        return false;
      }
    }
  }
  return true;
}

struct F8Args {
  F8Scales sa, sw;
  int M, N, K;
  int tiles_m, tiles_n;
  EpiParams ep;
};

// ---- epilogue ---------------------------------------------------------------------------------------------------
// An epilogue warp owns 32 rows x 64 columns, copied out of tensor memory into 64 registers a lane (one row each).  The
// small per-column operands live in the lanes, lane l holding columns l and 32 + l, and are passed around by shuffles:
// 16-byte loads per row and step, as the bf16 kernel does them, took 48 more registers, and the spills went through L2
// (shared memory leaves no L1): 8 100 cycles a tile against 2 600 now.  ACT is a template argument because eight unrolled
// steps with every activation's code in each of them do not fit the instruction cache.
constexpr int F8_COLS = EPI_BOX_COLS;
struct F8Cols {
  float bias[2], gate[2];
  bool per_row;  // the 32 rows belong to more than one batch element: gates are read row by row
};
__device__ __forceinline__ float f8_bf16(const void* p, int64_t i) { return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]); }

__device__ __forceinline__ F8Cols f8_cols(const EpiParams& ep, int m_box, int M, int64_t nbase, int64_t N, int lane) {
  F8Cols c;
  const int64_t b0 = m_box / ep.rows_per_batch;
  c.per_row = ep.gate_table != nullptr && (min(m_box + 31, M - 1) / ep.rows_per_batch) != b0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t n = nbase + 32 * j + lane;
    const bool in = n < N && m_box < M;
    c.bias[j] = ep.bias && in ? f8_bf16(ep.bias, n) : 0.f;
    c.gate[j] = ep.gate_table && in ? f8_bf16(ep.gate_table, ep.gate_row * N + n) + f8_bf16(ep.gate_t, (b0 * 6 + ep.gate_row) * N + n) : 0.f;
  }
  return c;
}

template <int ACT>
__device__ __forceinline__ bool f8_drain(EpiBox& eb, const F8Cols& cols, const EpiParams& ep, const uint32_t (&acc)[4][16], bool use_res,
                                         bool rows_in, int lane, int m_box, int M, int64_t nbase, int64_t N, const CUtensorMap* tmOut,
                                         volatile int* abort_flag) {
  if (nbase >= N) return true;  // uniform
  if (use_res) {
    if (!f8_wait(eb.res_bar, eb.res_phase, abort_flag, 5)) return false;
    eb.res_phase ^= 1u;
  }
  const bool has_bias = ep.bias != nullptr, has_gate = ep.gate_table != nullptr;
#pragma unroll
  for (int c = 0; c < 8; ++c) {  // 8 columns = 16 bytes of the row; N is a multiple of 8
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(acc[c >> 1][8 * (c & 1) + e]);
    if (has_bias) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += __shfl_sync(0xffffffffu, cols.bias[c >> 2], (8 * c + e) & 31);
    }
    if (ACT == 1) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fast_silu(v[e]);
    } else if (ACT == 2) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (nbase + 8 * c + e < ep.relu_cols) v[e] = v[e] < 0.f ? 0.f : v[e];
    } else if (ACT == 3) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = gelu_tanh(v[e]);
    }
    if (has_gate) {
      if (cols.per_row) {  // rare: out of line, one element at a time
        const int64_t b = min(m_box + lane, M - 1) / ep.rows_per_batch;
        for (int e = 0; e < 8; ++e) {
          const int64_t n = min(nbase + 8 * c + e, N - 1);
          const float g = f8_bf16(ep.gate_table, ep.gate_row * N + n) + f8_bf16(ep.gate_t, (b * 6 + ep.gate_row) * N + n);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = i == e ? v[i] * g : v[i];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= __shfl_sync(0xffffffffu, cols.gate[c >> 2], (8 * c + e) & 31);
      }
    }
    uint4* slot = reinterpret_cast<uint4*>(eb.row_g + (((uint32_t)c ^ eb.swz) << 4));
    if (use_res) {
      float f[8];
      unpack8(*slot, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += f[e];
    }
    *slot = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0 && rows_in) {
    tma_store_2d(tmOut, eb.box_s, (int)nbase, m_box);
    bulk_commit();
  }
  return true;
}

// start of a tile: once the previous tile's store has read the box, the residual is fetched into it
__device__ __forceinline__ void f8_box_begin(const EpiBox& eb, bool use_res, int lane, int m_box, int64_t nbase, int64_t N,
                                             const CUtensorMap* tmRes) {
  if (lane == 0) {
    bulk_wait_read_all();
    if (use_res && nbase < N) {
      mbar_expect_tx(eb.res_bar, (uint32_t)EPI_BOX_BYTES);
      tma_load_2d(eb.box_s, tmRes, eb.res_bar, (int)nbase, m_box);
    }
  }
  __syncwarp();
}

// ---- one CTA per 128 x 128 tile ---------------------------------------------------------------------------------
constexpr int S8_BM = 128, S8_BN = 128;
constexpr int S8_A_BYTES = S8_BM * 128, S8_B_BYTES = S8_BN * 128;
constexpr int S8_STAGE_BYTES = S8_A_BYTES + S8_B_BYTES;  // 32 KiB
constexpr int S8_STAGES = 5;
constexpr int S8_EPI_BYTES = F8_EPI_WARPS * EPI_BOX_BYTES;
constexpr int S8_SF_BYTES = 2 * 2 * 512;                 // two buffers of (A tile, W tile)
constexpr int S8_SMEM_BYTES = S8_STAGES * S8_STAGE_BYTES + S8_EPI_BYTES + S8_SF_BYTES + F8_CTRL_BYTES;
constexpr int S8_SF_COL0 = 2 * S8_BN;
static_assert(S8_SMEM_BYTES <= 232448, "shared memory budget");
static_assert(16 * S8_STAGES + 40 + 8 * F8_EPI_WARPS + 32 <= F8_CTRL_BYTES, "control block too small");

template <int ACT>
__global__ void __launch_bounds__(F8_THREADS, 1)
gemm_fp8_tc_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmRes, const F8Args args) {
  constexpr int STAGES = S8_STAGES;
  constexpr uint32_t IDESC = f8_idesc(S8_BM, S8_BN);
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t tiles_base = smem_u32(smem_raw);
  const uint32_t epi_base = tiles_base + STAGES * S8_STAGE_BYTES;
  unsigned char* epi_gen = smem_raw + STAGES * S8_STAGE_BYTES;
  const uint32_t sf_base = epi_base + S8_EPI_BYTES;
  unsigned char* sf_gen = epi_gen + S8_EPI_BYTES;
  const uint32_t ctrl = sf_base + S8_SF_BYTES;
  unsigned char* ctrl_gen = sf_gen + S8_SF_BYTES;
  // control: full[STAGES] | empty[STAGES] | tfull[2] | tempty[2] | tmem ptr | abort | res[EPI_WARPS] | sf[2] | sfempty[2]
  const uint32_t bar_full = ctrl, bar_empty = ctrl + 8 * STAGES;
  const uint32_t bar_tfull = ctrl + 16 * STAGES, bar_tempty = bar_tfull + 16;
  const uint32_t bar_res = ctrl + 16 * STAGES + 40;
  const uint32_t bar_sf = bar_res + 8 * F8_EPI_WARPS, bar_sfempty = bar_sf + 16;
  volatile uint32_t* tmem_ptr_slot = reinterpret_cast<volatile uint32_t*>(ctrl_gen + 16 * STAGES + 32);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl_gen + 16 * STAGES + 36);

  if ((tiles_base & 1023u) != 0u) {
    if (threadIdx.x == 0) atomicExch(&g_fp8_status, 9);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_tiles = args.tiles_m * args.tiles_n;
  const int kblocks = (args.K + F8_BK - 1) / F8_BK;
  const int kgroups = (kblocks + F8_GROUP - 1) / F8_GROUP;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(bar_tfull + 8 * a, 1);
      mbar_init(bar_tempty + 8 * a, F8_EPI_WARPS);
      mbar_init(bar_sf + 8 * a, 1);
      mbar_init(bar_sfempty + 8 * a, 1);
    }
    for (int w = 0; w < F8_EPI_WARPS; ++w) mbar_init(bar_res + 8 * w, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmOut) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmRes) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ctrl + 16 * STAGES + 32), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_ptr_slot;

  if (warp == 0) {
    // ------------------------------- loads --------------------------------------------
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
        const int mt = tile / args.tiles_n, nt = tile % args.tiles_n;
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!f8_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, 1)) { ok = false; break; }
          const uint32_t sa = tiles_base + stage * S8_STAGE_BYTES;
          const uint32_t fb = bar_full + 8 * stage;
          mbar_expect_tx(fb, S8_STAGE_BYTES);
          tma_load_2d(sa, &tmA, fb, kb * F8_BK, mt * S8_BM);
          tma_load_2d(sa + S8_A_BYTES, &tmB, fb, kb * F8_BK, nt * S8_BN);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------- MMA issuer ---------------------------------------
    // the warp waits together and one elected lane issues (see elect_one)
    uint32_t stage = 0, phase = 0, acc_phase = 0u, grp = 0;
    bool ok = true;
    int it = 0;
    auto wait = [&](uint32_t bar, uint32_t parity, int code) { return __all_sync(0xffffffffu, f8_wait(bar, parity, abort_flag, code)); };
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x, ++it) {
      const int a = it & 1;
      if (!wait(bar_tempty + 8 * a, ((acc_phase >> a) & 1u) ^ 1u, 2)) break;
      acc_phase ^= 1u << a;
      const uint32_t d_tmem = tmem_base + (uint32_t)(a * S8_BN);
      for (int kb = 0; kb < kblocks; ++kb) {
        const uint32_t buf = grp & 1u;
        if ((kb & (F8_GROUP - 1)) == 0 && !wait(bar_sf + 8 * buf, (grp >> 1) & 1u, 6)) { ok = false; break; }
        if (!wait(bar_full + 8 * stage, phase, 3)) { ok = false; break; }
        tcgen05_fence_after();
        const bool last = (kb & (F8_GROUP - 1)) == F8_GROUP - 1 || kb + 1 == kblocks;
        if (elect_one()) {
          const uint32_t sa = tiles_base + stage * S8_STAGE_BYTES;
          const uint64_t adesc = make_smem_desc(sa), bdesc = make_smem_desc(sa + S8_A_BYTES);
          const uint32_t sfa_t = tmem_base + (uint32_t)S8_SF_COL0 + 8 * buf, sfb_t = sfa_t + 4;
          const uint32_t idesc = IDESC | f8_scale_byte((uint32_t)(kb & (F8_GROUP - 1)));
#pragma unroll
          for (int k = 0; k < 4; ++k)  // 32 elements = 32 bytes inside the 128-byte swizzle row
            umma_fp8(d_tmem, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), idesc, sfa_t, sfb_t, (kb | k) != 0 ? 1u : 0u);
          umma_commit(bar_empty + 8 * stage);
          if (last) umma_commit(bar_sfempty + 8 * buf);
          if (kb + 1 == kblocks) umma_commit(bar_tfull + 8 * a);
        }
        __syncwarp();
        if (last) ++grp;
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 2) {
    // ------------------------------- scale tiles --------------------------------------
    uint32_t grp = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
      const int m0 = (tile / args.tiles_n) * S8_BM, n0 = (tile % args.tiles_n) * S8_BN;
      uint4 wa = f8_scale_words(args.sa, m0, 0, lane), wb = f8_scale_words(args.sw, n0, 0, lane);
      for (int g = 0; g < kgroups; ++g, ++grp) {
        const uint32_t buf = grp & 1u, ph = (grp >> 1) & 1u;
        const uint4 ca = wa, cb = wb;
        if (g + 1 < kgroups) {  // the next tile's words are in flight during this one's wait
          wa = f8_scale_words(args.sa, m0, g + 1, lane);
          wb = f8_scale_words(args.sw, n0, g + 1, lane);
        }
        // the MMAs that used this buffer are done, and so is the copy that read the shared tile
        if (!f8_wait(bar_sfempty + 8 * buf, ph ^ 1u, abort_flag, 7)) ok = false;
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        unsigned char* t = sf_gen + buf * 1024 + lane * 16;
        *reinterpret_cast<uint4*>(t) = ca;
        *reinterpret_cast<uint4*>(t + 512) = cb;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tcgen05_fence_after();
          const uint32_t sfa_t = tmem_base + (uint32_t)S8_SF_COL0 + 8 * buf;
          tmem_cp_sf(sfa_t, make_sf_desc(sf_base + buf * 1024));
          tmem_cp_sf(sfa_t + 4, make_sf_desc(sf_base + buf * 1024 + 512));
          umma_commit(bar_sf + 8 * buf);
        }
        __syncwarp();
      }
    }
  } else if (warp >= 4) {
    // ------------------------------- epilogue warps -----------------------------------
    const int ew = warp - 4;
    const int quad = warp & 3;
    const int half = ew >> 2;
    static_assert(S8_BN == 2 * F8_COLS, "two warps share a row of the tile");
    const EpiParams& ep = args.ep;
    const int64_t N = args.N;
    const bool has_res = ep.residual != nullptr;
    EpiBox eb;
    eb.box_s = epi_base + (uint32_t)(ew * EPI_BOX_BYTES);
    eb.row_g = epi_gen + ew * EPI_BOX_BYTES + lane * 128;
    eb.res_bar = bar_res + 8 * ew;
    eb.res_phase = 0u;
    eb.swz = (uint32_t)(lane & 7);
    uint32_t full_phase = 0u;
    int it = 0;
    for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x, ++it) {
      const int a = it & 1;
      const int m_box = (tile / args.tiles_n) * S8_BM + quad * 32;
      const int64_t nbase = (int64_t)(tile % args.tiles_n) * S8_BN + half * F8_COLS;
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(a * S8_BN + half * F8_COLS);
      const bool rows_in = m_box < args.M, use_res = has_res && rows_in;
      f8_box_begin(eb, use_res, lane, m_box, nbase, N, &tmRes);
      const F8Cols cols = f8_cols(ep, m_box, args.M, nbase, N, lane);
      if (!f8_wait(bar_tfull + 8 * a, (full_phase >> a) & 1u, abort_flag, 4)) break;
      full_phase ^= 1u << a;
      tcgen05_fence_after();
      uint32_t acc[4][16];
      epi_acc_load<4>(taddr, acc);
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_tempty + 8 * a);
      if (!f8_drain<ACT>(eb, cols, ep, acc, use_res, rows_in, lane, m_box, args.M, nbase, N, &tmOut, abort_flag)) break;
    }
    if (lane == 0) bulk_wait_all();
  }

  __syncwarp();
  if (*abort_flag) {  // give copies and products in flight time to end before shared and tensor memory are released
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) {}
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// ---- CTA pairs on 256 x 256 tiles -------------------------------------------------------------------------------
// Each CTA of a cluster of two loads its own 128 rows of A and half of the W tile; the leader issues the MMAs
// (cta_group::2, M = 256).  Tensor memory holds one 256-column accumulator and the scale tiles, so the epilogue warps
// copy the accumulator into registers, hand it back and finish under the next tile's MMAs (as in the NVFP4 kernel).
// Both CTAs build the scale tiles of their own A rows and of the whole W tile in their own shared memory; the leader
// is told when both are there (bar_sfready counts two arrivals) and issues the copies for both.
constexpr int P8_BM = 128, P8_BN = 256;
constexpr int P8_A_BYTES = P8_BM * 128, P8_B_BYTES = (P8_BN / 2) * 128;
constexpr int P8_STAGE_BYTES = P8_A_BYTES + P8_B_BYTES;  // 32 KiB
constexpr int P8_STAGES = 5;
constexpr int P8_EPI_WARPS = 16;                         // four per tensor-memory quadrant, 64 columns (one box) each
constexpr int P8_THREADS = 128 + 32 * P8_EPI_WARPS;
constexpr int P8_EPI_BYTES = P8_EPI_WARPS * EPI_BOX_BYTES;
constexpr int P8_CTRL_BYTES = 512;
constexpr int P8_SF_TILE = 3 * 512;                      // A rows, W rows 0..127, W rows 128..255
constexpr int P8_SF_BYTES = P8_SF_TILE;                   // one: a copy takes far less than the four stages it serves
constexpr int P8_SMEM_BYTES = P8_STAGES * P8_STAGE_BYTES + P8_EPI_BYTES + P8_SF_BYTES + P8_CTRL_BYTES;
constexpr int P8_SF_COL0 = P8_BN, P8_SF_COLS = 12;
static_assert(P8_SMEM_BYTES <= 232448, "shared memory budget");
static_assert(16 * P8_STAGES + 40 + 8 * P8_EPI_WARPS + 48 <= P8_CTRL_BYTES, "control block too small");

template <int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(P8_THREADS, 1)
gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                     const __grid_constant__ CUtensorMap tmOut, const __grid_constant__ CUtensorMap tmRes, const F8Args args) {
  constexpr int STAGES = P8_STAGES;
  constexpr uint32_t IDESC = f8_idesc(256, P8_BN);
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t tiles_base = smem_u32(smem_raw);
  const uint32_t epi_base = tiles_base + STAGES * P8_STAGE_BYTES;
  unsigned char* epi_gen = smem_raw + STAGES * P8_STAGE_BYTES;
  const uint32_t sf_base = epi_base + P8_EPI_BYTES;
  unsigned char* sf_gen = epi_gen + P8_EPI_BYTES;
  const uint32_t ctrl = sf_base + P8_SF_BYTES;
  unsigned char* ctrl_gen = sf_gen + P8_SF_BYTES;
  // control: full[STAGES] | empty[STAGES] | tfull | pad | tempty | pad | tmem ptr | abort | res[EPI_WARPS] | sf[2] |
  // sfempty[2] | sfready[2]
  const uint32_t bar_full = ctrl, bar_empty = ctrl + 8 * STAGES;
  const uint32_t bar_tfull = ctrl + 16 * STAGES, bar_tempty = bar_tfull + 16;
  const uint32_t bar_res = ctrl + 16 * STAGES + 40;
  const uint32_t bar_sf = bar_res + 8 * P8_EPI_WARPS, bar_sfempty = bar_sf + 16, bar_sfready = bar_sf + 32;
  volatile uint32_t* tmem_ptr_slot = reinterpret_cast<volatile uint32_t*>(ctrl_gen + 16 * STAGES + 32);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctrl_gen + 16 * STAGES + 36);

  if ((tiles_base & 1023u) != 0u) {  // cluster-uniform: the dynamic window starts at the same offset in every CTA
    if (threadIdx.x == 0) atomicExch(&g_fp8_status, 9);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1;
  const int num_tiles = args.tiles_m * args.tiles_n;
  const int kblocks = (args.K + F8_BK - 1) / F8_BK;
  const int kgroups = (kblocks + F8_GROUP - 1) / F8_GROUP;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full + 8 * s, 1);
      mbar_init(bar_empty + 8 * s, 1);
    }
    mbar_init(bar_tfull, 1);
    mbar_init(bar_tempty, 2 * P8_EPI_WARPS);
    for (int a = 0; a < 2; ++a) {
      mbar_init(bar_sf + 8 * a, 1);
      mbar_init(bar_sfempty + 8 * a, 1);
      mbar_init(bar_sfready + 8 * a, 2);
    }
    for (int w = 0; w < P8_EPI_WARPS; ++w) mbar_init(bar_res + 8 * w, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmOut) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmRes) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ctrl + 16 * STAGES + 32), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers are initialised before anything signals them
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_ptr_slot;
  if (warp == 0) {
    // ------------------------------- loads (both CTAs) ----------------------------------
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      const uint32_t full0 = map_to_cta(bar_full, 0);
      for (int tile = cluster_id; tile < num_tiles && ok; tile += num_clusters) {
        int mt, nt;
        pair_tile_coords(tile, args.tiles_m, args.tiles_n, mt, nt);
        const int m0 = mt * 256 + (int)rank * P8_BM;
        const int n0 = nt * P8_BN + (int)rank * (P8_BN / 2);
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!f8_wait(bar_empty + 8 * stage, phase ^ 1u, abort_flag, 1)) { ok = false; break; }
          const uint32_t sa = tiles_base + stage * P8_STAGE_BYTES;
          if (leader) mbar_expect_tx(bar_full + 8 * stage, 2 * P8_STAGE_BYTES);
          const uint32_t fb = full0 + 8 * stage;
          tma_load_2d_pair(sa, &tmA, fb, kb * F8_BK, m0);
          tma_load_2d_pair(sa + P8_A_BYTES, &tmB, fb, kb * F8_BK, n0);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------- MMA issuer (leader CTA only) -----------------------
    if (leader) {
      uint32_t stage = 0, phase = 0, acc_phase = 0, grp = 0;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity, int code) { return __all_sync(0xffffffffu, f8_wait(bar, parity, abort_flag, code)); };
      for (int tile = cluster_id; tile < num_tiles && ok; tile += num_clusters) {
        if (!wait(bar_tempty, acc_phase ^ 1u, 2)) break;
        acc_phase ^= 1u;
        for (int kb = 0; kb < kblocks; ++kb) {
          const uint32_t buf = grp & 1u;
          if ((kb & (F8_GROUP - 1)) == 0 && !wait(bar_sf + 8 * buf, (grp >> 1) & 1u, 6)) { ok = false; break; }
          if (!wait(bar_full + 8 * stage, phase, 3)) { ok = false; break; }
          tcgen05_fence_after();
          const bool last = (kb & (F8_GROUP - 1)) == F8_GROUP - 1 || kb + 1 == kblocks;
          if (elect_one()) {
            const uint32_t sa = tiles_base + stage * P8_STAGE_BYTES;
            const uint64_t adesc = make_smem_desc(sa), bdesc = make_smem_desc(sa + P8_A_BYTES);
            const uint32_t sfa_t = tmem_base + (uint32_t)P8_SF_COL0 + P8_SF_COLS * buf, sfb_t = sfa_t + 4;
            const uint32_t idesc = IDESC | f8_scale_byte((uint32_t)(kb & (F8_GROUP - 1)));
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_fp8_pair(tmem_base, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), idesc, sfa_t, sfb_t,
                            (kb | k) != 0 ? 1u : 0u);
            umma_commit_pair(bar_empty + 8 * stage);  // frees this stage in both CTAs
            if (last) tc_commit_pair_local(bar_sfempty + 8 * buf);
            if (kb + 1 == kblocks) umma_commit_pair(bar_tfull);  // accumulator complete, both CTAs
          }
          __syncwarp();
          if (last) ++grp;
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp == 2) {
    // ------------------------------- scale tiles (both CTAs build, the leader copies) ----
    uint32_t grp = 0;
    bool ok = true;
    const uint32_t ready0 = map_to_cta(bar_sfready, 0);
    for (int tile = cluster_id; tile < num_tiles && ok; tile += num_clusters) {
      int mt, nt;
      pair_tile_coords(tile, args.tiles_m, args.tiles_n, mt, nt);
      const int m0 = mt * 256 + (int)rank * P8_BM, n0 = nt * P8_BN;
      uint4 wa = f8_scale_words(args.sa, m0, 0, lane), wb = f8_scale_words(args.sw, n0, 0, lane),
            wc = f8_scale_words(args.sw, n0 + 128, 0, lane);
      for (int g = 0; g < kgroups; ++g, ++grp) {
        const uint32_t buf = grp & 1u, ph = (grp >> 1) & 1u;
        // the copies that read the shared tiles of the group before are done (one commit tells both CTAs)
        if (grp > 0 && !f8_wait(bar_sf + 8 * (buf ^ 1u), ((grp - 1) >> 1) & 1u, abort_flag, 8)) ok = false;
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        unsigned char* t = sf_gen + lane * 16;
        *reinterpret_cast<uint4*>(t) = wa;
        *reinterpret_cast<uint4*>(t + 512) = wb;
        *reinterpret_cast<uint4*>(t + 1024) = wc;
        fence_proxy_async_smem();
        __syncwarp();
        if (g + 1 < kgroups) {  // in flight while the leader waits and copies
          wa = f8_scale_words(args.sa, m0, g + 1, lane);
          wb = f8_scale_words(args.sw, n0, g + 1, lane);
          wc = f8_scale_words(args.sw, n0 + 128, g + 1, lane);
        }
        if (lane == 0) {
          mbar_arrive_cluster(ready0 + 8 * buf);
          if (leader) {
            if (!f8_wait(bar_sfready + 8 * buf, ph, abort_flag, 9)) ok = false;
            // the MMAs that used this buffer's columns are done
            if (ok && !f8_wait(bar_sfempty + 8 * buf, ph ^ 1u, abort_flag, 7)) ok = false;
            if (ok) {
              tcgen05_fence_after();
              const uint32_t sfa_t = tmem_base + (uint32_t)P8_SF_COL0 + P8_SF_COLS * buf;
              tmem_cp_sf_pair(sfa_t, make_sf_desc(sf_base));
              tmem_cp_sf_pair(sfa_t + 4, make_sf_desc(sf_base + 512));
              tmem_cp_sf_pair(sfa_t + 8, make_sf_desc(sf_base + 1024));
              umma_commit_pair(bar_sf + 8 * buf);
            }
          }
        }
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      }
    }
  } else if (warp >= 4) {
    // ------------------------------- epilogue warps (both CTAs) -------------------------
    const int ew = warp - 4;
    const int quad = warp & 3;
    const int part = ew >> 2;
    static_assert(4 * F8_COLS == P8_BN, "four warps share a row of the tile");
    const EpiParams& ep = args.ep;
    const int64_t N = args.N;
    const bool has_res = ep.residual != nullptr;
    const uint32_t tempty0 = map_to_cta(bar_tempty, 0);
    EpiBox eb;
    eb.box_s = epi_base + (uint32_t)(ew * EPI_BOX_BYTES);
    eb.row_g = epi_gen + ew * EPI_BOX_BYTES + lane * 128;
    eb.res_bar = bar_res + 8 * ew;
    eb.res_phase = 0u;
    eb.swz = (uint32_t)(lane & 7);
    uint32_t full_phase = 0u;
    for (int tile = cluster_id; tile < num_tiles; tile += num_clusters) {
      int mt, nt;
      pair_tile_coords(tile, args.tiles_m, args.tiles_n, mt, nt);
      const int m_box = mt * 256 + (int)rank * P8_BM + quad * 32;
      const int64_t nbase = (int64_t)nt * P8_BN + part * F8_COLS;
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(part * F8_COLS);
      const bool rows_in = m_box < args.M, use_res = has_res && rows_in;
      f8_box_begin(eb, use_res, lane, m_box, nbase, N, &tmRes);
      const F8Cols cols = f8_cols(ep, m_box, args.M, nbase, N, lane);
      if (!f8_wait(bar_tfull, full_phase, abort_flag, 4)) break;
      full_phase ^= 1u;
      tcgen05_fence_after();
      uint32_t acc[4][16];
      epi_acc_load<4>(taddr, acc);
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tempty0);
      if (!f8_drain<ACT>(eb, cols, ep, acc, use_res, rows_in, lane, m_box, args.M, nbase, N, &tmOut, abort_flag)) break;
    }
    if (lane == 0) bulk_wait_all();
  }

  __syncwarp();
  if (*abort_flag) {  // give copies and products in flight time to end before shared and tensor memory are released
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) {}
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();  // nobody leaves while the other CTA may still signal or read it
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// ---- a few rows (single tokens): the weight is streamed once --------------------------------------------------------
// Bound by the bytes of W and, at these sizes, by one trip to memory: 1 x 2240 -> 6720 (15 MB) 6.5 us, 2.3 TB/s, where the
// copy rate would allow 2.3 us.  A CTA takes 16 of its rows, its warps split the 128-blocks of K, every load of a warp is
// 16 bytes and issued before the first is needed.  mma.sync with the W rows as M and the tokens as N (8 a tile): the
// contraction index may be permuted as long as both operands agree, so a lane's 16 contiguous bytes of a row are the
// fragments of two instructions.  A block's sum is scaled by 2^(ea + ew) in fp32 and added; the warps' sums meet in
// shared memory in a fixed order.
__device__ __forceinline__ void mma_e4m3_16832(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d * 2^(e + f - 254), e and f E8M0 bytes (255: NaN): in two factors, so that neither leaves the range of fp32
__device__ __forceinline__ float f8_scaled(float d, int e, int f) {
  const int s = e + f, h = s >> 1;
  return d * __uint_as_float(max(e, f) == 255 ? 0x7fffffffu : (uint32_t)h << 23) * __uint_as_float((uint32_t)(s - h) << 23);
}

template <int NT8, int WARPS>
__global__ void __launch_bounds__(32 * WARPS) gemm_fp8_rows_kernel(const unsigned char* __restrict__ A, const unsigned char* __restrict__ W,
                                                            __nv_bfloat16* __restrict__ out, int64_t ldo, const F8Args args) {
  __shared__ float4 red[WARPS][NT8][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int n0 = blockIdx.x * 16, K = args.K, kblocks = (K + 127) / 128;
  const int r0 = n0 + g, r1 = n0 + g + 8;
  const bool in0 = r0 < args.N, in1 = r1 < args.N;
  const unsigned char *w0 = W + (int64_t)(in0 ? r0 : 0) * K, *w1 = W + (int64_t)(in1 ? r1 : 0) * K;
  const unsigned char *s0 = args.sw.p + ((in0 ? r0 : 0) >> args.sw.shift) * args.sw.ld, *s1 = args.sw.p + ((in1 ? r1 : 0) >> args.sw.shift) * args.sw.ld;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  float acc[NT8][4] = {};
#pragma unroll 2
  for (int kb = warp; kb < kblocks; kb += WARPS) {
    const int k = kb * 128 + 16 * c;
    const bool ka = k < K, kz = k + 64 < K;  // K is a multiple of 16
    const uint4 wa0 = in0 && ka ? ldg_nc_u4(w0 + k) : zero, wa1 = in1 && ka ? ldg_nc_u4(w1 + k) : zero;
    const uint4 wz0 = in0 && kz ? ldg_nc_u4(w0 + k + 64) : zero, wz1 = in1 && kz ? ldg_nc_u4(w1 + k + 64) : zero;
    const int e0 = __ldg(s0 + kb), e1 = __ldg(s1 + kb);
#pragma unroll
    for (int t = 0; t < NT8; ++t) {
      const int m = 8 * t + g;
      const bool min_ = m < args.M;
      const unsigned char* x = A + (int64_t)(min_ ? m : 0) * K + k;
      const uint4 xa = min_ && ka ? __ldg(reinterpret_cast<const uint4*>(x)) : zero;
      const uint4 xz = min_ && kz ? __ldg(reinterpret_cast<const uint4*>(x + 64)) : zero;
      float d[4] = {0.f, 0.f, 0.f, 0.f};
      mma_e4m3_16832(d, wa0.x, wa1.x, wa0.y, wa1.y, xa.x, xa.y);
      mma_e4m3_16832(d, wa0.z, wa1.z, wa0.w, wa1.w, xa.z, xa.w);
      mma_e4m3_16832(d, wz0.x, wz1.x, wz0.y, wz1.y, xz.x, xz.y);
      mma_e4m3_16832(d, wz0.z, wz1.z, wz0.w, wz1.w, xz.z, xz.w);
      const int ma = 8 * t + 2 * c, mb = ma + 1;
      const int f0 = ma < args.M ? __ldg(args.sa.p + (ma >> args.sa.shift) * args.sa.ld + kb) : 127;
      const int f1 = mb < args.M ? __ldg(args.sa.p + (mb >> args.sa.shift) * args.sa.ld + kb) : 127;
      acc[t][0] += f8_scaled(d[0], e0, f0);
      acc[t][1] += f8_scaled(d[1], e0, f1);
      acc[t][2] += f8_scaled(d[2], e1, f0);
      acc[t][3] += f8_scaled(d[3], e1, f1);
    }
  }
#pragma unroll
  for (int t = 0; t < NT8; ++t) red[warp][t][lane] = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * 8 * NT8; i += 32 * WARPS) {
    const int r = i & 15, m = i >> 4;  // W row of the CTA, token
    if (m >= args.M || n0 + r >= args.N) continue;
    const int from = (r & 7) * 4 + ((m & 7) >> 1), word = (r >> 3) * 2 + (m & 1);
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += reinterpret_cast<const float*>(&red[w][m >> 3][from])[word];
    out[(int64_t)m * ldo + n0 + r] = from_f32<__nv_bfloat16>(epi_scalar<__nv_bfloat16>(v, m, n0 + r, args.N, args.ep));
  }
}

// ---- quantiser --------------------------------------------------------------------------------------------------
// The least e with amax <= 448 * 2^e (448 = 1.75 * 2^8), from the bits of amax: exponent - 8, one more when the
// fraction is above 1.75; at least -126 (which a block of zeros takes).  Returns the E8M0 byte e + 127.
__device__ __forceinline__ uint32_t f8_scale_of(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(max(e, -126) + 127);
}
// 2^-e for the byte e + 127, which lies in [1, 247] (the largest fp32 value takes e = 120)
__device__ __forceinline__ float f8_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float f8_finite_abs(float x) {  // |x|, or 0 for an infinity or NaN
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}
// two values -> two E4M3 codes; a non-finite value becomes NaN (the conversion alone would saturate an infinity)
__device__ __forceinline__ uint32_t f8_codes2(float lo, float hi, float inv) {
  const float nan = __uint_as_float(0x7fffffffu);
  lo = fabsf(lo) <= 3.402823466e38f ? lo * inv : nan;
  hi = fabsf(hi) <= 3.402823466e38f ? hi * inv : nan;
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// Largest finite magnitude of 8 elements.
__device__ __forceinline__ float f8_amax8(const float (&f)[8]) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = fmaxf(m, f8_finite_abs(f[e]));
  return m;
}
__device__ __forceinline__ uint2 f8_codes8(const float (&f)[8], float inv) {
  return make_uint2(f8_codes2(f[0], f[1], inv) | (f8_codes2(f[2], f[3], inv) << 16),
                    f8_codes2(f[4], f[5], inv) | (f8_codes2(f[6], f[7], inv) << 16));
}
// The same on packed bf16: magnitudes compare as integers, and only a vector that holds an infinity or NaN (bits of at
// least 0x7f80) takes the general form.
__device__ __forceinline__ uint32_t f8_packed_max(const uint4& v) {
  const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
  return max(m & 0xffffu, m >> 16);
}
__device__ __forceinline__ uint32_t f8_codes2_finite(uint32_t pair, float inv) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(bf16_lo(pair) * inv, bf16_hi(pair) * inv), __NV_SATFINITE, __NV_E4M3);
}

template <typename T>
__device__ __forceinline__ void f8_load8(const T* p, float (&f)[8]);
template <>
__device__ __forceinline__ void f8_load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&f)[8]) { unpack8(ldg_nc_u4(p), f); }
template <>
__device__ __forceinline__ void f8_load8<float>(const float* p, float (&f)[8]) {
  const uint4 a = ldg_nc_u4(p), b = ldg_nc_u4(p + 4);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(w[e]);
}

// Bound by HBM (2 or 4 bytes read, 1 written per element): 16384 x 5600 bf16 47-51 us, 5.4-5.8 TB/s, up to 0.89 of the copy
// rate; fp32 77 us, 5.9 TB/s.
// One scale for each row and 128 elements: 8 lanes hold a block, 16 elements each (with 16 lanes the maximum's shuffles, the
// scale and the addresses cost as many instructions as the conversion, and their issue bound the kernel: 56 us), of R rows
// at a time (their loads are in flight together; R = 1 where there are few rows, so that more CTAs share the work).
template <typename T, int R>
__global__ void __launch_bounds__(256) fp8_quantize_rows_kernel(const T* __restrict__ x, int64_t ld, unsigned char* __restrict__ q,
                                                                unsigned char* __restrict__ sf, int64_t ldsf, int64_t rows, int K,
                                                                int kblocks) {
  const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 3;  // (group of R rows, block)
  const int sub = threadIdx.x & 7;
  const uint32_t group = (uint32_t)unit / (uint32_t)kblocks;  // the host keeps the units below 2^31
  const int64_t r0 = (int64_t)group * R;
  if (r0 >= rows) return;  // 8 lanes leave together
  const int kb = (int)((uint32_t)unit - group * (uint32_t)kblocks);
  const int k = kb * 128 + 16 * sub;
  const bool in = k < K;  // K is a multiple of 16
  const uint32_t eight = 0xffu << (threadIdx.x & 24);
  const T* xr = x + r0 * ld + k;
  unsigned char* qr = q + r0 * K + k;
  unsigned char* sr = sf + r0 * ldsf + kb;
  auto emit = [&](int i, float m, auto codes) {  // row r0 + i: the block's maximum, its scale, this lane's codes
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(eight, m, o));
    const uint32_t byte = f8_scale_of(m);
    if (sub == 0) sr[i * ldsf] = (unsigned char)byte;
    if (in) {
      const float inv = f8_inverse(byte);
      const uint2 c = codes(0, inv), d = codes(1, inv);
      *reinterpret_cast<uint4*>(qr + (int64_t)i * K) = make_uint4(c.x, c.y, d.x, d.y);
    }
  };
  if constexpr (sizeof(T) == 2) {
    uint4 v[R][2];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        v[i][h] = in && r0 + i < rows ? ldg_nc_u4(xr + i * ld + 8 * h) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (r0 + i >= rows) break;  // the same for the 8 lanes
      const uint32_t m = max(f8_packed_max(v[i][0]), f8_packed_max(v[i][1]));
      const bool finite = m < 0x7f80u;
      float f[2][8], amax = __uint_as_float(m << 16);
      if (!finite) {
        unpack8(v[i][0], f[0]);
        unpack8(v[i][1], f[1]);
        amax = fmaxf(f8_amax8(f[0]), f8_amax8(f[1]));
      }
      emit(i, amax, [&](int h, float inv) {
        if (!finite) return f8_codes8(f[h], inv);
        return make_uint2(f8_codes2_finite(v[i][h].x, inv) | (f8_codes2_finite(v[i][h].y, inv) << 16),
                          f8_codes2_finite(v[i][h].z, inv) | (f8_codes2_finite(v[i][h].w, inv) << 16));
      });
    }
  } else {
    float f[R][2][8];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i][h][e] = 0.f;
        if (in && r0 + i < rows) f8_load8(xr + i * ld + 8 * h, f[i][h]);
      }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (r0 + i >= rows) break;
      emit(i, fmaxf(f8_amax8(f[i][0]), f8_amax8(f[i][1])), [&](int h, float inv) { return f8_codes8(f[i][h], inv); });
    }
  }
}

// One scale for each 128 x 128 block (weights, quantised once): a CTA per block, rows in 8 passes of 16.  16384 x 5600 bf16
// 81 us, fp32 102: all of a CTA's loads come before its one rendezvous, all of its stores after; made once a weight.
template <typename T>
__global__ void __launch_bounds__(256) fp8_quantize_tiles_kernel(const T* __restrict__ x, int64_t ld, unsigned char* __restrict__ q,
                                                                 unsigned char* __restrict__ sf, int64_t ldsf, int64_t rows, int K) {
  __shared__ float red[8];
  const int sub = threadIdx.x & 15, slot = threadIdx.x >> 4;
  const int k = blockIdx.x * 128 + 8 * sub;
  const int64_t r0 = (int64_t)blockIdx.y * 128;
  float f[8][8];
  float m = 0.f;
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int64_t r = r0 + 16 * p + slot;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[p][e] = 0.f;
    if (k < K && r < rows) f8_load8(x + r * ld + k, f[p]);
    m = fmaxf(m, f8_amax8(f[p]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, red[w]);
  const uint32_t byte = f8_scale_of(m);
  if (threadIdx.x == 0) sf[blockIdx.y * ldsf + blockIdx.x] = (unsigned char)byte;
  const float inv = f8_inverse(byte);
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int64_t r = r0 + 16 * p + slot;
    if (k < K && r < rows)
      *reinterpret_cast<uint2*>(q + r * K + k) = f8_codes8(f[p], inv);
  }
}

template <typename T>
static int launch_quantize(const void* x, int64_t ld, void* q, void* sf, int64_t ldsf, int64_t rows, int64_t K, int block_rows,
                           cudaStream_t st) {
  const int64_t kblocks = ceil_div(K, 128);
  const T* xp = static_cast<const T*>(x);
  unsigned char *qp = static_cast<unsigned char*>(q), *sp = static_cast<unsigned char*>(sf);
  if (block_rows == 1) {
    constexpr int R = 2;
    const int64_t most = (int64_t)1 << 31;
    SANA_REQUIRE(ceil_div(rows, R) * kblocks < most, "sana_fp8_quantize: too large");
    if (ceil_div(rows, R) * kblocks >= 32 * 8 * (int64_t)sm_count())  // eight CTAs per SM are left with R rows each
      fp8_quantize_rows_kernel<T, R><<<(unsigned)ceil_div(ceil_div(rows, R) * kblocks, 32), 256, 0, st>>>(xp, ld, qp, sp, ldsf, rows,
                                                                                                         (int)K, (int)kblocks);
    else
      fp8_quantize_rows_kernel<T, 1><<<(unsigned)ceil_div(rows * kblocks, 32), 256, 0, st>>>(xp, ld, qp, sp, ldsf, rows, (int)K,
                                                                                          (int)kblocks);
  } else {
    const int64_t rb = ceil_div(rows, 128);
    SANA_REQUIRE(rb <= 65535, "sana_fp8_quantize: more than 65535 blocks of 128 rows");
    fp8_quantize_tiles_kernel<T><<<dim3((unsigned)kblocks, (unsigned)rb), 256, 0, st>>>(xp, ld, qp, sp, ldsf, rows, (int)K);
  }
  SANA_LAUNCH_CHECK("fp8_quantize kernel");
  return SANA_OK;
}

// Most rows the streaming kernel takes: at M = 16 it needs 3.7 - 12.3 us where the tile kernel needs 7.3 - 18 (K x N from
// 1152 x 1152 to 2240 x 11200); at 24 rows 17 against 10.5 us (2240 x 6720).
constexpr int64_t F8_ROWS = 16;

template <int ACT>
static int launch_gemm_fp8(bool pair, const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmOut,
                           const CUtensorMap& tmRes, F8Args& a, cudaStream_t st) {
  a.tiles_m = (int)ceil_div(a.M, pair ? 256 : S8_BM);
  a.tiles_n = (int)ceil_div(a.N, pair ? P8_BN : S8_BN);
  const int64_t tiles = (int64_t)a.tiles_m * a.tiles_n;
  SANA_REQUIRE(tiles < ((int64_t)1 << 30), "sana_gemm_fp8: too many tiles");
  static OncePerDevice once;
  if (auto first = once.first_time()) {
    cudaError_t e = cudaFuncSetAttribute(gemm_fp8_pair_kernel<ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, P8_SMEM_BYTES);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(gemm_fp8_tc_kernel<ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S8_SMEM_BYTES);
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(gemm_fp8)");
  }
  if (pair) {
    const int64_t max_clusters = sm_count() / 2;
    const int grid = (int)(2 * (tiles < max_clusters ? tiles : max_clusters));
    gemm_fp8_pair_kernel<ACT><<<grid, P8_THREADS, P8_SMEM_BYTES, st>>>(tmA, tmB, tmOut, tmRes, a);
  } else {
    const int grid = (int)(tiles < sm_count() ? tiles : sm_count());
    gemm_fp8_tc_kernel<ACT><<<grid, F8_THREADS, S8_SMEM_BYTES, st>>>(tmA, tmB, tmOut, tmRes, a);
  }
  SANA_LAUNCH_CHECK("gemm_fp8 kernel");
  return SANA_OK;
}

}  // namespace sana

using namespace sana;

extern "C" int sana_fp8_quantize(const void* x, int64_t ld, void* q, void* sf, int64_t ldsf, int64_t rows, int64_t K,
                                 int block_rows, int dtype, void* stream) {
  SANA_REQUIRE(x && q && sf, "sana_fp8_quantize: null pointer");
  SANA_REQUIRE(rows > 0 && K > 0 && K % 16 == 0 && K < ((int64_t)1 << 30), "sana_fp8_quantize: K must be a positive multiple of 16");
  SANA_REQUIRE(block_rows == 1 || block_rows == 128, "sana_fp8_quantize: block_rows must be 1 or 128");
  SANA_REQUIRE(dtype == SANA_BF16 || dtype == SANA_F32, "sana_fp8_quantize: unknown dtype %d", dtype);
  SANA_REQUIRE(ld >= K && ld % (dtype == SANA_BF16 ? 8 : 4) == 0, "sana_fp8_quantize: ld must be >= K and keep rows 16-byte aligned");
  SANA_REQUIRE(ldsf >= ceil_div(K, 128), "sana_fp8_quantize: ldsf too small");
  SANA_REQUIRE(rows < ((int64_t)1 << 31), "sana_fp8_quantize: too many rows");
  SANA_REQUIRE(aligned16(x) && aligned16(q), "sana_fp8_quantize: alignment");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == SANA_BF16 ? launch_quantize<__nv_bfloat16>(x, ld, q, sf, ldsf, rows, K, block_rows, st)
                            : launch_quantize<float>(x, ld, q, sf, ldsf, rows, K, block_rows, st);
}

extern "C" int sana_gemm_fp8(const void* Aq, const void* sfa, int64_t ldsfa, int a_block_rows, const void* Wq, const void* sfw,
                             int64_t ldsfw, int w_block_rows, void* out, int64_t ldo, int64_t M, int64_t N, int64_t K,
                             const sana_gemm_epilogue* ep, void* stream) {
  SANA_REQUIRE(Aq && sfa && Wq && sfw && out, "sana_gemm_fp8: null pointer");
  SANA_REQUIRE(M > 0 && N > 0 && K > 0, "sana_gemm_fp8: M, N, K must be positive");
  SANA_REQUIRE(K % 16 == 0 && N % 8 == 0 && ldo >= N && ldo % 8 == 0, "sana_gemm_fp8: K %% 16, N %% 8, ldo %% 8 required");
  SANA_REQUIRE(M < ((int64_t)1 << 31) - 256 && N < ((int64_t)1 << 31) - 256 && K < ((int64_t)1 << 30), "sana_gemm_fp8: size out of range");
  SANA_REQUIRE((a_block_rows == 1 || a_block_rows == 128) && (w_block_rows == 1 || w_block_rows == 128),
               "sana_gemm_fp8: block_rows must be 1 or 128");
  const int64_t words = ceil_div(ceil_div(K, 128), 4) * 4;
  SANA_REQUIRE(ldsfa >= words && ldsfw >= words && ldsfa % 4 == 0 && ldsfw % 4 == 0 &&
                   (reinterpret_cast<uintptr_t>(sfa) & 3) == 0 && (reinterpret_cast<uintptr_t>(sfw) & 3) == 0,
               "sana_gemm_fp8: scale rows must be 4-byte aligned and padded to a multiple of 4 blocks");
  SANA_REQUIRE(aligned16(Aq) && aligned16(Wq) && aligned16(out), "sana_gemm_fp8: alignment");
  EpiParams p;
  int rc = check_epilogue(ep, N, &p, "sana_gemm_fp8");
  if (rc) return rc;
  SANA_REQUIRE(!p.residual || (aligned16(p.residual) && p.ldr % 8 == 0), "sana_gemm_fp8: residual alignment");
  SANA_REQUIRE(!p.bias || aligned16(p.bias), "sana_gemm_fp8: bias alignment");
  SANA_REQUIRE(!p.gate_table || (aligned16(p.gate_table) && aligned16(p.gate_t)), "sana_gemm_fp8: gate alignment");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  F8Args a;
  a.sa = {static_cast<const unsigned char*>(sfa), ldsfa, M, a_block_rows == 128 ? 7 : 0};
  a.sw = {static_cast<const unsigned char*>(sfw), ldsfw, N, w_block_rows == 128 ? 7 : 0};
  a.M = (int)M, a.N = (int)N, a.K = (int)K;
  a.ep = p;
  if (M <= F8_ROWS && gemm_variant() == 0) {
    const unsigned char *ap = static_cast<const unsigned char*>(Aq), *wp = static_cast<const unsigned char*>(Wq);
    __nv_bfloat16* op = static_cast<__nv_bfloat16*>(out);
    const unsigned grid = (unsigned)ceil_div(N, 16);
    // 16 warps a CTA while every CTA has an SM of its own (M = 1: N = 1152 3.2 us against 4.2 with eight, N = 2240, K = 5600
    // 6.8 against 9.0); eight beyond, where several share one (N = 6720 6.5 against 9.1, N = 11200 9.8 against 12.6)
    const bool wide = ceil_div(N, 16) <= sm_count();
    if (M <= 8 && wide) gemm_fp8_rows_kernel<1, 16><<<grid, 512, 0, st>>>(ap, wp, op, ldo, a);
    else if (M <= 8) gemm_fp8_rows_kernel<1, 8><<<grid, 256, 0, st>>>(ap, wp, op, ldo, a);
    else if (wide) gemm_fp8_rows_kernel<2, 16><<<grid, 512, 0, st>>>(ap, wp, op, ldo, a);
    else gemm_fp8_rows_kernel<2, 8><<<grid, 256, 0, st>>>(ap, wp, op, ldo, a);
    SANA_LAUNCH_CHECK("gemm_fp8_rows kernel");
    return SANA_OK;
  }
  CUtensorMap tmA, tmB, tmOut, tmRes;
  rc = make_tmap_2d(&tmOut, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, out, M, N, ldo * 2, 32, EPI_BOX_COLS);
  if (rc) return rc;
  tmRes = tmOut;
  if (p.residual) {
    rc = make_tmap_2d(&tmRes, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.residual, M, N, p.ldr * 2, 32, EPI_BOX_COLS);
    if (rc) return rc;
  }
  const int variant = gemm_variant();
  const bool pair = variant == 2 || (variant == 0 && M >= 2048);
  rc = make_tmap_2d(&tmA, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, Aq, M, K, K, 128, F8_BK);
  if (rc) return rc;
  rc = make_tmap_2d(&tmB, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, Wq, N, K, K, 128, F8_BK);
  if (rc) return rc;
  switch (p.act) {
    case 0: return launch_gemm_fp8<0>(pair, tmA, tmB, tmOut, tmRes, a, st);
    case 1: return launch_gemm_fp8<1>(pair, tmA, tmB, tmOut, tmRes, a, st);
    case 2: return launch_gemm_fp8<2>(pair, tmA, tmB, tmOut, tmRes, a, st);
    default: return launch_gemm_fp8<3>(pair, tmA, tmB, tmOut, tmRes, a, st);
  }
}

extern "C" int sana_gemm_fp8_take_device_status(int* status_out) {
  if (!status_out) return fail(SANA_ERR_INVALID, "sana_gemm_fp8_take_device_status: null pointer");
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_fp8_status, sizeof(int));
  if (e != cudaSuccess) return cuda_status(e, "cudaMemcpyFromSymbol(g_fp8_status)");
  if (v != 0) {
    int zero = 0;
    e = cudaMemcpyToSymbol(g_fp8_status, &zero, sizeof(int));
    if (e != cudaSuccess) return cuda_status(e, "cudaMemcpyToSymbol(g_fp8_status)");
  }
  *status_out = v;
  return SANA_OK;
}
