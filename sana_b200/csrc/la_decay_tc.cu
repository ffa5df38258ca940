// Causal linear attention with a decay for each head, bf16, on the 5th-generation tensor cores (formulas in la_decay.cu).
//
// A CTA walks one token segment of one head in chunks of 128 tokens.  With v1 = [v ; 1] (the ones column makes the key sum
// and the normaliser come out of the same products), w_t = lambda^(C-1-t), and S the state before the chunk:
//
//   scores  SC  = phi(Q) phi(K)^T                     M = 128 queries, N = 128 keys, K = D
//   inter   O1  = phi(Q) S^T                          N = D + 16, K = D          row t is scaled by lambda^(t+1) at the end
//   intra   O2  = (SC * lambda^(t-s), s <= t) V       N = D, K = 128             A operand in tensor memory, two bf16 terms
//   state   dS^T = (w K)^T V1                         M = D key channels, N = D + 16, K = 128 tokens
//
// Every tile is [64-channel block][row][128 bytes], 128-byte swizzled, which serves as a K-major operand (rows = M or N)
// and as an MN-major one (rows = K) alike: k and q are stored once and used both ways, and the bulk-tensor copies write
// them in place (4-D views (channel, head, token, sample): channels past the head arrive as zeros).
//
// Roles: warps 0-3 keep the state (thread j: key channel j against all value channels, fp32 registers), join the chunk's
// sum to it (S = lambda^C S + dS: one rounded multiply-add per chunk, since the tensor core truncates its sums), write it
// as the bf16 operand of O1, and finish the outputs; warps 4-7 decay and mask the scores; the next 4 or 8 warps weight the
// keys, apply ReLU in place and put the ones column back beside v; one warp issues the products, one the copies.
// The weighted k is split into NT bf16 terms: 3 where the state leaves the kernel (2^-24; the truncation of a chunk's 24
// products adds up to 2e-6 where everything has one sign and nothing decays, 3e-7 otherwise), 2 where it only serves the
// outputs (2^-17, below their own rounding).  Up to 32 channels the terms stand side by side in the 128
// rows of one product, and the state warps add them: an instruction costs the same (elect_one) whatever part of its rows
// is used.  The decayed scores enter O2 as two bf16 terms (2^-17; heads of 128 channels: the last 64 keys of a chunk as
// one, 2^-8), which costs 1-3 % of the time: an output of a few tokens would feel one rounding of a score as much as its
// own.  The carried key sum enters O1 as two terms, the state's value channels as two or one (write_operand).  All waits
// are bounded.
//
// Measured (L2 flushed before each run): 20 heads of 112 channels, 16 384 tokens 159 us (1.85 TB/s of q, k, v, out; the copy
// rate would allow 45); 8 x 4096 tokens, 70 heads of 32 246-254 us (2.4 TB/s; 90); 8 x 4096 tokens, 16 heads of 128 288 us
// (two launches; 83); 4 x up to 4096, 16 heads of 64 over 8 of k and v 63-86.  What bounds it is the length of a chunk's
// chain - copy, transform, products, join, state operand, products, output, each behind a barrier and with one warp per
// scheduler for each role: the tensor pipe is busy 20-27 % of the time and DRAM 25-38 %.  Chunks of 128 halve the number of
// chains that 64 would have, and two CTAs of narrow heads per SM overlap theirs; wide heads fill shared memory alone.
// Single-lane waits (half the speed of converged ones) and roles that poll several barriers in turn were tried and were
// slower.
#include "la_decay.cuh"

namespace sana {

__device__ int g_ld_status = 0;

constexpr int LT_C = 128;
constexpr int LT_BLK = LT_C * 128;  // one 64-channel block of a token tile

template <int D, int NT, bool OUT>
struct Lt {
  static constexpr int NV = D + 16;                      // value columns: D channels, the ones column, padding
  static constexpr int KB = (D + 63) / 64, VB = (NV + 63) / 64;
  static constexpr int LW = D <= 64 ? 4 : 8;             // warps that weight the keys: thread = token (and half of its channels)
  static constexpr int LT = 32 * LW;
  static constexpr bool WIDE = D >= 80;
  static constexpr int THREADS = 32 * (8 + LW + (WIDE ? 4 : 2));  // wide heads: whole warpgroups, for the register split
  static constexpr bool STACK = D <= 32;                 // terms of the weighted k side by side, 32 channels apart
  static constexpr int MMAS = STACK ? 1 : NT;            // products per 16 tokens of the state update
  static constexpr int KTILE = KB * LT_BLK, VTILE = VB * LT_BLK;
  static constexpr int WTILE = STACK ? 2 * LT_BLK : NT * KTILE;
  static constexpr int STATE_BLK = D * 128;              // bf16 state operand: rows = key channels
  static constexpr int X_BYTES = STACK ? (D + 1) * 32 * (NT == 3 ? 10 : 8) : 0;  // sums of the terms, [D+1][32]; the third in bf16
  static constexpr int SCRATCH = (OUT ? VB * STATE_BLK : 0) + X_BYTES + 4 * (32 + LT_C + 2 + 32) + (OUT ? 4 * 2 * LT_C : 0) + 248 +
                                 4 * (4 + 4 * D);
  static constexpr int ONE_EACH = WTILE + VTILE + KTILE + (OUT ? KTILE : 0) + SCRATCH;
  static constexpr int LIMIT = OUT && D <= 32 ? 113 * 1024 : 232448;  // two CTAs per SM, or one
  // a second v tile hides the latency of its load behind the products that still need the first; then one for q
  static constexpr int VBUF = ONE_EACH + VTILE <= LIMIT ? 2 : 1;
  static constexpr int QBUF = OUT && ONE_EACH + (VBUF - 1) * VTILE + KTILE <= LIMIT ? 2 : 1;
  // Terms of the state operand: a second one where there is room for it beside these (16, 48 and 64 channels).  With no decay
  // to speak of it takes the outputs' error from 2.2e-3 to 1.7e-3, and costs 2 % (16 channels), 11 % (8 x 4096 tokens, 40
  // heads of 48: 336 -> 373 us), 5-9 % (4 x up to 4096, 16 heads of 64).
  static constexpr int ST = OUT && ONE_EACH + (VBUF - 1) * VTILE + (QBUF - 1) * KTILE + VB * STATE_BLK <= LIMIT ? 2 : 1;
  static constexpr int OFF_W = 0;                        // weighted k (followed by v: with one block of 64 channels, rows
  static constexpr int OFF_V = OFF_W + WTILE;            // 64 .. 127 of the product read there and are not used)
  static constexpr int OFF_K = OFF_V + VBUF * VTILE;
  static constexpr int OFF_Q = OFF_K + KTILE;
  static constexpr int OFF_S = OFF_Q + (OUT ? QBUF * KTILE : 0);
  static constexpr int OFF_X = OFF_S + (OUT ? ST * VB * STATE_BLK : 0);
  static constexpr int OFF_POW = OFF_X + X_BYTES;        // powers behind 32 zeros
  static constexpr int OFF_RS = OFF_POW + 4 * (32 + LT_C + 2 + 32);  // row sums of the scores, [2][128]
  static constexpr int OFF_BAR = OFF_RS + (OUT ? 4 * 2 * LT_C : 0);
  // Tokens whose v is not finite, by channel, for the last chunks: a flag each, then the first such token (128: none).
  static constexpr int BADS = VBUF == 2 ? 4 : 2;  // a chunk's entries are cleared before the one BADS later can be filled
  // Barriers, then the tensor-memory address and the abort flag.  With one v tile its second barriers are free, and one of
  // them does for bready (128 channels leave no room for another).
  static constexpr int BARS = VBUF == 2 ? 30 : 29;
  static constexpr int OFF_SLOT = OFF_BAR + 8 * BARS;
  static constexpr int OFF_BAD = OFF_SLOT + 8;
  static constexpr int BYTES = OFF_BAD + 4 * (BADS + BADS * D);
  // Scores in two halves of 64 keys.  O2 has columns of its own, except for 128 channels, where it starts inside the
  // second half and the next chunk's scores wait until it has been read.
  static constexpr bool ALIAS = 128 + 2 * NV + D > 512;
  static constexpr int COL_SC = 0, COL_O2 = ALIAS ? 96 : 128;
  // The decayed scores of 32 keys go over their fp32 scores, which have been read: 16 columns of bf16 pairs, and 16 of what
  // that rounding left.  Where O2 starts at 96, the last 64 keys have room for the first term only.
  __host__ __device__ static constexpr bool two_terms(int blk) { return !ALIAS || blk < 2; }
  __host__ __device__ static constexpr int pair_col(int blk) { return COL_SC + (two_terms(blk) ? 32 * blk : 64 + 16 * (blk - 2)); }
  static constexpr int COL_O1 = COL_O2 + D;
  static constexpr int COL_DS = OUT ? COL_O1 + NV : 0;
  static constexpr int COLS = COL_DS + NV;
  static constexpr int TMEM_COLS = COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
  // arrivals that complete a phase of barrier i (their order: at the top of the kernel); kempty, without scores: k is free
  // once the LW warps have weighted it
  __host__ __device__ static constexpr int arrivals(int i) {
    return !OUT && i == 5 ? LW : VBUF == 1 && i == 7 ? 4 : i < 17 ? 1 : i < 19 ? LW / 2 : i < 22 ? LW : 4;
  }
  static constexpr int CTAS = TMEM_COLS <= 256 && 2 * (BYTES + 1024) <= 228 * 1024 && D <= 32 ? 2 : 1;  // resident per SM
  // D = f32 (bit 4), A = B = bf16 (7, 10), transposes (MN-major) at 15 / 16, N >> 3 at 17, M >> 4 at 24
  static constexpr uint32_t BASE = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24);
  static constexpr uint32_t ID_SC = BASE | ((64u >> 3) << 17);
  static constexpr uint32_t ID_O1 = BASE | (1u << 16) | ((uint32_t)(NV >> 3) << 17);
  static constexpr uint32_t ID_O2 = BASE | (1u << 16) | ((uint32_t)(D >> 3) << 17);
  static constexpr uint32_t ID_DS = BASE | (1u << 15) | (1u << 16) | ((uint32_t)(NV >> 3) << 17);
  static_assert(COLS <= 512 && BYTES <= 232448, "budgets");
};

__device__ __forceinline__ uint64_t lt_desc_mn(uint32_t saddr, uint32_t block_stride_bytes) {
  const uint32_t lo = ((saddr >> 4) & 0x3FFFu) | ((block_stride_bytes >> 4) << 16);
  const uint32_t hi = (1024u >> 4) | (1u << 14) | (2u << 29);
  return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ void lt_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Nothing that uses these registers may move above the wait for the loads that fill them, while others are under way.
__device__ __forceinline__ void lt_arrived(uint32_t (&r)[16]) {
  asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
               "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void lt_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ uint32_t lt_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr) : "memory");
  return r;
}

// whether a phase is complete, without waiting
__device__ __forceinline__ bool lt_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// Bounded wait like mbar_wait, by all lanes of a warp and with the plain poll: the suspend hint of mbar_wait puts the warp
// to sleep in steps, up to a microsecond past the arrival, and a chunk passes through eight waits in a row.
__device__ __forceinline__ bool lt_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait_poll(bar, parity))) return true;
  const long long t0 = clock64();
  uint32_t spins = 0;
  while (!__all_sync(0xffffffffu, mbar_try_wait_poll(bar, parity))) {
    if ((++spins & 255u) == 0) {
      bool stop = *abort_flag != 0;
      if (!stop && clock64() - t0 > TC_WAIT_LIMIT_CYCLES) {
        *abort_flag = code;
        atomicExch(&g_ld_status, code);
        stop = true;
      }
      if (__any_sync(0xffffffffu, stop)) return false;
    }
  }
  return true;
}

// whether all of the four state warps say so: a barrier of 128 threads
__device__ __forceinline__ bool lt_all(bool mine) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.and.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r) : "r"((uint32_t)mine) : "memory");
  return r != 0;
}

template <int D, int NT, bool OUT>
__global__ void __launch_bounds__(Lt<D, NT, OUT>::THREADS, Lt<D, NT, OUT>::CTAS) 
la_decay_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const __grid_constant__ CUtensorMap tmQ, const LdArgs a) {
  using T = Lt<D, NT, OUT>;
  constexpr int C = LT_C, NV = T::NV, LW = T::LW;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t sm = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if ((sm & 1023u) != 0u) {  // uniform over the CTA: nothing has been set up yet
    if (tid == 0) atomicExch(&g_ld_status, 9);
    return;
  }
  float* pow_s = reinterpret_cast<float*>(smem + T::OFF_POW) + 32;  // pow_s[n] = lambda^n, 0 for n in [-32, -1]
  // barriers: raw tiles have landed / tiles are ready (weighted k: by halves of 64 tokens) / tiles are free; scores ready,
  // decayed scores ready, chunk sum ready / read, state operand ready / read, outputs ready / read
  const uint32_t bar = sm + T::OFF_BAR;
  // (a pair is indexed by the half of the tokens or keys, or by the buffer, so that no wait can be two phases late)
  const uint32_t kraw = bar, vraw = bar + 8 /* 2 */, qraw = bar + 24 /* 2 */, kempty = bar + 40, vempty = bar + 48 /* 2 */;
  const uint32_t qempty = bar + 64 /* 2 */, wempty = bar + 80 /* 2 */, scready = bar + 96 /* 2 */, dsready = bar + 112;
  const uint32_t sopread = bar + 120, oready = bar + 128;                                        // 17 of one arrival
  const uint32_t wfull = bar + 136 /* 2 */, vfull = bar + 152, qfull = bar + 160, kfull = bar + 168;
  const uint32_t pready = bar + 176 /* 2 */, rsready = bar + 192 /* 2 */, dsread = bar + 208, sopready = bar + 216, oread = bar + 224;
  const uint32_t bready = T::VBUF == 2 ? bar + 232 : vempty + 8;  // the state warps have looked at a chunk's non-finite v
  const uint32_t slot = sm + T::OFF_SLOT;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + T::OFF_SLOT);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + T::OFF_SLOT + 4);

  const int h = blockIdx.x, seg = blockIdx.y, b = blockIdx.z;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.N) : a.N;
  const int seg_begin = seg * a.seg_len, seg_end = min(a.N, seg_begin + a.seg_len);
  const int n_begin = min(seg_begin, len), n_end = min(seg_end, len);
  const int chunks = (n_end - n_begin + C - 1) / C;
  const float gl = a.log_decay[h];
  const int64_t row0 = (int64_t)b * a.N;
  const int64_t per = (int64_t)(D + 1) * D;

  if (tid == 0) {
    for (int i = 0; i < T::BARS; ++i) mbar_init(bar + 8 * i, T::arrivals(i));
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"((uint32_t)T::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  int* bad_flag = reinterpret_cast<int*>(smem + T::OFF_BAD);
  int* bad_from = bad_flag + T::BADS;
  for (int i = tid; i < T::BADS + T::BADS * D; i += T::THREADS) bad_flag[i] = i < T::BADS ? 0 : C;
  for (int i = tid - 32; i <= C; i += T::THREADS) pow_s[i] = i < 0 ? 0.f : ld_power(gl, i);
  float* rev_s = pow_s + C + 2;  // lambda^(31 - k)
  if (tid < 32) rev_s[tid] = ld_power(gl, 31 - tid);
  // the ones column of v1 and its padding, once: token t, channels D .. D + 15 = two 16-byte pieces
  for (int i = tid; i < 2 * C * T::VBUF; i += T::THREADS) {
    const int t = (i >> 1) % C, ch = D / 8 + (i & 1);
    *reinterpret_cast<uint4*>(smem + T::OFF_V + i / (2 * C) * T::VTILE + (ch >> 3) * LT_BLK + t * 128 + (((ch & 7) ^ (t & 7)) << 4)) =
        make_uint4((i & 1) ? 0u : 0x3f80u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Wide heads: 640 threads start with 96 registers each; the state warps, which hold a row of the state, take over what
  // the others give up: 128 x 192 + 128 x 64 + 256 x 72 + 128 x 80 = 61 440 = 640 x 96
  if (warp < 4) {
    // ------------------------------- state and outputs ---------------------------------
    if constexpr (T::WIDE) asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const int j = tid;            // key channel (state)
    const int t = tid;            // query of the chunk (outputs)
    const bool jin = j < D, warp_in = warp * 32 < D;
    // Narrow heads: lane = key channel, warp w holds value channels 8 w .. + 7 and (warp 3) the key sum; else thread = key
    // channel holds all of them.
    constexpr int NS = T::STACK ? 9 : D + 1;
    const int sj = T::STACK ? lane : j;
    const bool sin = T::STACK ? lane < D : jin;
    auto row_of = [&](int i) -> int { return !T::STACK ? i : i == 8 ? D : 8 * warp + i; };
    auto held = [&](int i) -> bool { return !T::STACK || (i == 8 ? warp == 3 : 8 * warp < D); };
    float S[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) S[i] = 0.f;
    if (OUT && sin && (chunks > 0 || seg == a.nseg - 1)) {  // the state before this segment
      auto add = [&](const float* src, float f) {
#pragma unroll
        for (int i = 0; i < NS; ++i)
          if (held(i)) S[i] = fmaf(f, __ldg(src + row_of(i) * D + sj), S[i]);
      };
      if (a.prior) add(a.prior + ((int64_t)b * a.H + h) * per, ld_power(gl, n_begin));
      for (int r = 0; r < seg; ++r) {
        const int end = min((r + 1) * a.seg_len, len);
        if (end == min(r * a.seg_len, len)) break;  // past the sequence: these segments hold nothing
        add(a.partial + (((int64_t)b * a.npart + r) * a.H + h) * per, ld_power(gl, n_begin - end));
      }
      if (a.npart > 0 && seg == a.nseg - 1) {  // the exact sums of all segments are known: the state after the last token
        float* dst = a.state + ((int64_t)b * a.H + h) * per;
        const float* src = a.partial + (((int64_t)b * a.npart + seg) * a.H + h) * per;
        const float f = ld_power(gl, n_end - n_begin);
#pragma unroll
        for (int i = 0; i < NS; ++i)
          if (held(i)) dst[row_of(i) * D + sj] = fmaf(f, S[i], n_end > n_begin ? __ldg(src + row_of(i) * D + sj) : 0.f);
      }
    }
    // Row j of the state operand, 8 value channels to a 16-byte piece.  The value channels enter as two bf16 terms (2^-17) where
    // shared memory has room for a second operand, else as one (2^-8 of each at most, of either
    // sign, summed over D key channels).  The key sum, whose error all channels of an output would share, always enters
    // as two: the second takes a column of the padding.
    auto key_sum = [](float z) -> uint32_t { return pack_bf16(z, z - __bfloat162float(__float2bfloat16_rn(z))); };
    auto left2 = [](float a, float b, uint32_t w) -> uint32_t {
      const float2 d = __fadd2_rn(make_float2(a, b), make_float2(-bf16_lo(w), -bf16_hi(w)));
      return pack_bf16(d.x, d.y);
    };
    auto write_operand = [&]() {
      if constexpr (T::STACK) {
        unsigned char* row = smem + T::OFF_S + lane * 128;
        auto put = [&](int c, const uint4& w, int term = 0) {  // c < 8
          *reinterpret_cast<uint4*>(row + term * T::VB * T::STATE_BLK + ((c ^ (lane & 7)) << 4)) = w;
        };
        if (lane < D && 8 * warp < D) {
          const uint4 w = make_uint4(pack_bf16(S[0], S[1]), pack_bf16(S[2], S[3]), pack_bf16(S[4], S[5]), pack_bf16(S[6], S[7]));
          put(warp, w);
          if (T::ST == 2)
            put(warp, make_uint4(left2(S[0], S[1], w.x), left2(S[2], S[3], w.y), left2(S[4], S[5], w.z), left2(S[6], S[7], w.w)), 1);
        }
        if (lane < D && warp == 3) {
          put(D / 8, make_uint4(key_sum(S[8]), 0u, 0u, 0u));
          put(D / 8 + 1, make_uint4(0u, 0u, 0u, 0u));
          if (T::ST == 2) {
            put(D / 8, make_uint4(0u, 0u, 0u, 0u), 1);
            put(D / 8 + 1, make_uint4(0u, 0u, 0u, 0u), 1);
          }
        }
      } else if (jin) {
        unsigned char* row = smem + T::OFF_S + j * 128;
#pragma unroll
        for (int c = 0; c < NV / 8; ++c) {
          uint32_t w[4], r[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 8 * c + 2 * e;
            w[e] = i < D ? pack_bf16(S[i < D ? i : 0], S[i + 1 < D ? i + 1 : 0]) : i == D ? key_sum(S[NS - 1]) : 0u;
            r[e] = i < D ? left2(S[i < D ? i : 0], S[i + 1 < D ? i + 1 : 0], w[e]) : 0u;
          }
          unsigned char* at = row + (c >> 3) * T::STATE_BLK + (((c & 7) ^ (j & 7)) << 4);
          *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
          if (T::ST == 2) *reinterpret_cast<uint4*>(at + T::VB * T::STATE_BLK) = make_uint4(r[0], r[1], r[2], r[3]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(sopready);
    };
    if (OUT && chunks > 0) write_operand();
    bool ok = true;
    uint32_t bphase = 0u;
    for (int c = 0; c < chunks; ++c) {
      const uint32_t ph = (uint32_t)(c & 1);
      const int n0 = n_begin + c * C, nv = min(C, n_end - n0);
      ok = ok && lt_wait(dsready, ph, abort_flag, 1);
      tcgen05_fence_after();
      if constexpr (T::STACK) {  // warp s holds the sum of term s, lane = key channel: through shared memory, then warp by channels
        float* x = reinterpret_cast<float*>(smem + T::OFF_X) + lane;
        __nv_bfloat16* x3 = reinterpret_cast<__nv_bfloat16*>(smem + T::OFF_X + 2 * (D + 1) * 32 * 4) + lane;
        if (ok && warp < NT) {
          uint32_t d[NV];
#pragma unroll
          for (int g = 0; g < D / 16; ++g) tmem_ld_32x16(tmem + lanes + (uint32_t)(T::COL_DS + 16 * g), *reinterpret_cast<uint32_t(*)[16]>(d + 16 * g));
          d[D] = lt_ld1(tmem + lanes + (uint32_t)(T::COL_DS + D));
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i <= D; ++i) {
            if (warp < 2) x[(warp * (D + 1) + i) * 32] = __uint_as_float(d[i]);
            else x3[i * 32] = __float2bfloat16_rn(__uint_as_float(d[i]));  // 2^-16 of the first: its rounding is below 2^-24
          }
        }
        // The four warps go on or leave together.  A named barrier (an mbarrier cost 3 % more), which always fills:
        // whatever a warp's waits say, each of them ends, and nothing but this leaves the loop before its last chunk.
        ok = lt_all(ok);  // the scratch is free again once every warp has arrived at dsread
        if (!ok) break;
        const float whole = pow_s[nv];
#pragma unroll
        for (int i = 0; i < NS; ++i)
          if (held(i)) {
            float r = x[(D + 1 + row_of(i)) * 32];
            if (NT == 3) r += __bfloat162float(x3[row_of(i) * 32]);
            S[i] = fmaf(whole, S[i], x[row_of(i) * 32] + r);
          }
      } else if (!ok) {
        break;
      } else if (warp_in) {
        const float whole = pow_s[nv];
        uint32_t d[2][16];  // the next columns are under way while these are added
        tmem_ld_32x16(tmem + lanes + (uint32_t)T::COL_DS, d[0]);
        const uint32_t z = lt_ld1(tmem + lanes + (uint32_t)(T::COL_DS + D));
#pragma unroll
        for (int g = 0; g < D / 16; ++g) {
          tmem_ld_wait();
          lt_arrived(d[g & 1]);
          if (g + 1 < D / 16) tmem_ld_32x16(tmem + lanes + (uint32_t)(T::COL_DS + 16 * (g + 1)), d[(g + 1) & 1]);
#pragma unroll
          for (int e = 0; e < 16; ++e) S[16 * g + e] = fmaf(whole, S[16 * g + e], __uint_as_float(d[g & 1][e]));
        }
        S[NS - 1] = fmaf(whole, S[NS - 1], __uint_as_float(z));
      }
      volatile int* bad = bad_flag + c % T::BADS;
      const int* from = bad_from + c % T::BADS * D;
      const bool poisoned = OUT && *bad != 0;  // the same for the four warps: cleared behind their common barrier
      if (poisoned) {
#pragma unroll
        for (int i = 0; i < NS; ++i)
          if (held(i) && row_of(i) < D && from[row_of(i)] < C) S[i] = __uint_as_float(0x7fffffffu);
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dsread);
      if (OUT) {
        if (c + 1 < chunks) {
          if (!lt_wait(sopread, ph, abort_flag, 2)) { ok = false; continue; }
          write_operand();
        }
        if (!lt_wait(oready, ph, abort_flag, 3)) { ok = false; continue; }
        tcgen05_fence_after();
        const float f = pow_s[t + 1];
        float m = a.scale;
        if (a.normalise) {
          if (!lt_wait(rsready + 8 * ph, (uint32_t)(c >> 1) & 1u, abort_flag, 3)) { ok = false; continue; }
          const uint32_t d1 = lt_ld1(tmem + lanes + (uint32_t)(T::COL_O1 + D));      // q with the key sum: its first term,
          const uint32_t d2 = lt_ld1(tmem + lanes + (uint32_t)(T::COL_O1 + D + 1));  // its second
          tmem_ld_wait();
          m = 1.f / (fmaf(f, __uint_as_float(d1) + __uint_as_float(d2),
                          reinterpret_cast<const float*>(smem + T::OFF_RS)[(c & 1) * C + t]) + a.eps);
        }
        __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(a.out) + (row0 + n0 + t) * a.ldo + (int64_t)h * D;
        uint32_t x[16], y[16];
        tmem_ld_32x16(tmem + lanes + (uint32_t)T::COL_O1, x);
        tmem_ld_32x16(tmem + lanes + (uint32_t)T::COL_O2, y);
        tmem_ld_wait();
#pragma unroll 1
        for (int g = 0; g < D / 16; ++g) {
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 o = __fmul2_rn(ffma2(make_float2(f, f), make_float2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])),
                                              make_float2(__uint_as_float(y[2 * e]), __uint_as_float(y[2 * e + 1]))),
                                        make_float2(m, m));
            w[e] = pack_bf16(o.x, o.y);
          }
          if (g + 1 < D / 16) {  // the next columns are under way while these are stored
            tmem_ld_32x16(tmem + lanes + (uint32_t)(T::COL_O1 + 16 * (g + 1)), x);
            tmem_ld_32x16(tmem + lanes + (uint32_t)(T::COL_O2 + 16 * (g + 1)), y);
          }
          if (poisoned) {
            for (int e = 0; e < 16; ++e)
              if (t >= from[16 * g + e]) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  if (k == e >> 1) w[k] |= (e & 1) ? 0x7fff0000u : 0x00007fffu;
              }
          }
          if (t < nv) {
            if (a.wide_rows) {  // 32-byte aligned rows: whole sectors
              asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + 16 * g), "r"(w[0]), "r"(w[1]),
                           "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
            } else {
              *reinterpret_cast<uint4*>(dst + 16 * g) = make_uint4(w[0], w[1], w[2], w[3]);
              *reinterpret_cast<uint4*>(dst + 16 * g + 8) = make_uint4(w[4], w[5], w[6], w[7]);
            }
          }
          tmem_ld_wait();
          lt_arrived(x);
          lt_arrived(y);
        }
        if (poisoned) {
          __syncwarp();
          if (lane == 0) mbar_arrive(bready);
          if (!lt_wait(bready, bphase, abort_flag, 21)) { ok = false; continue; }
          bphase ^= 1u;
          for (int i = tid; i < D; i += 128) bad_from[c % T::BADS * D + i] = C;
          if (tid == 0) *bad = 0;
          __threadfence_block();
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(oread);
      }
    }
    if (ok && sin && (!OUT || (a.npart == 0 && seg == a.nseg - 1))) {
      float* dst = OUT ? a.state + ((int64_t)b * a.H + h) * per : a.partial + (((int64_t)b * a.npart + seg) * a.H + h) * per;
#pragma unroll
      for (int i = 0; i < NS; ++i)
        if (held(i)) dst[row_of(i) * D + sj] = S[i];
    }
  } else if (warp < 8) {
    // ------------------------------- scores --------------------------------------------
    if constexpr (T::WIDE) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (OUT) {
      const int w = warp - 4;
      const uint32_t sc = tmem + ((uint32_t)(w * 32) << 16) + (uint32_t)T::COL_SC;
      float* rs = reinterpret_cast<float*>(smem + T::OFF_RS) + 32 * w + lane;
      const float* mine = pow_s + lane;
      for (int c = 0; c < chunks; ++c) {
        float2 sum = make_float2(0.f, 0.f);
        bool ok = true;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {  // rolled: four roles share the instruction cache
          if (!lt_wait(scready + 8 * half, (uint32_t)(c & 1), abort_flag, 4)) { ok = false; break; }
          tcgen05_fence_after();
#pragma unroll 1
          for (int q = 0; q < 2; ++q) {  // keys 32 blk .. + 31
            const int blk = 2 * half + q;
            uint32_t p[16], r[16];  // the first terms, the second ones
            auto split = [&](int e, const float2 v) {
              sum = __fadd2_rn(sum, v);
              p[e] = pack_bf16(v.x, v.y);
              const float2 left = __fadd2_rn(v, make_float2(-bf16_lo(p[e]), -bf16_hi(p[e])));
              r[e] = pack_bf16(left.x, left.y);
            };
            if (blk > w) {
#pragma unroll
              for (int e = 0; e < 16; ++e) p[e] = r[e] = 0u;
            } else {
              uint32_t x[32];
              tmem_ld_32x32(sc + (uint32_t)(32 * blk), x);
              tmem_ld_wait();
              if (blk < w) {  // every key lies before every query: lambda^(t - s) = lambda^(t - s0 - 31) lambda^(31 - k)
                const float f = mine[32 * (w - blk) - 31];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  const float2 d = __fmul2_rn(make_float2(f, f), *reinterpret_cast<const float2*>(rev_s + 2 * e));
                  split(e, __fmul2_rn(make_float2(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), d));
                }
              } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) {  // selected, not multiplied by the table's zero: a later token may be NaN
                  split(e, __fmul2_rn(make_float2(lane >= 2 * e ? __uint_as_float(x[2 * e]) : 0.f,
                                                  lane >= 2 * e + 1 ? __uint_as_float(x[2 * e + 1]) : 0.f),
                                      make_float2(mine[-2 * e], mine[-2 * e - 1])));
                }
              }
            }
            const uint32_t at = sc + (uint32_t)(T::pair_col(blk) - T::COL_SC);
            lt_st16(at, p);
            if (T::two_terms(blk)) lt_st16(at + 16, r);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          if (half == 1 && a.normalise) rs[(c & 1) * C] = sum.x + sum.y;
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(pready + 8 * half);
            if (half == 1 && a.normalise) mbar_arrive(rsready + 8 * (c & 1));
          }
        }
        if (!ok) break;
      }
      // rows of the segment past the sequence are zeros
      const int z0 = max(seg_begin, n_end);
      for (int64_t i = tid - 128; i < (int64_t)max(0, seg_end - z0) * (D / 8); i += 128) {
        const int t = z0 + (int)(i / (D / 8)), ch = (int)(i % (D / 8));
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + (row0 + t) * a.ldo + (int64_t)h * D + 8 * ch) =
            make_uint4(0u, 0u, 0u, 0u);
      }
    }
  } else if (warp < 8 + LW) {
    // ------------------------------- weighted keys, features, ones column ----------------
    if constexpr (T::WIDE) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    const int row = (tid - 256) & 127, part = (tid - 256) >> 7;  // token of the chunk; which of the interleaved 16-byte pieces
    constexpr int PARTS = T::LT / 128;
    const bool relu = a.relu != 0;
    const uint32_t wbar = 8u * (uint32_t)(row >> 6);  // warp-uniform: the half of the tokens
    unsigned char* krow = smem + T::OFF_K + row * 128;
    unsigned char* qrow = smem + T::OFF_Q + row * 128;
    unsigned char* vrow = smem + T::OFF_V + row * 128;
    auto piece = [&](int ch) -> uint32_t { return (uint32_t)((ch >> 3) * LT_BLK + (((ch & 7) ^ (row & 7)) << 4)); };
    // Outputs must not see an infinity or NaN in v before its token (below).  Where a first launch has summed the segment, one
    // key channel of that sum tells whether there is any; the sum itself is right to be NaN.
    bool look = OUT;
    if (OUT && a.npart > 0) {
      const float* src = a.partial + (((int64_t)b * a.npart + seg) * a.H + h) * per;
      bool odd = false;
      for (int i = lane; i < D; i += 32) odd |= !(fabsf(__ldg(src + i * D)) <= 3.402823466e38f);
      look = __any_sync(0xffffffffu, odd);
    }
    auto relu4 = [&](uint4 r) { return make_uint4(ld_relu2(r.x), ld_relu2(r.y), ld_relu2(r.z), ld_relu2(r.w)); };
    auto publish = [&](uint32_t full) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
    };
    for (int c = 0; c < chunks; ++c) {
      const uint32_t ph = (uint32_t)(c & 1);
      const int nv = min(C, n_end - (n_begin + c * C));
      const bool live = row < nv;
      constexpr int PIECES = D / 8 / PARTS;
      // features first: the next scores need them, the weights only when the state's products of the chunk before are done
      if (!lt_wait(kraw, ph, abort_flag, 5)) break;
      uint4 r[PIECES];
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        r[i] = *reinterpret_cast<const uint4*>(krow + piece(i * PARTS + part));
        if (relu) {
          r[i] = relu4(r[i]);
          if (OUT) *reinterpret_cast<uint4*>(krow + piece(i * PARTS + part)) = r[i];
        }
      }
      if constexpr (OUT) {
        publish(kfull);
        if (!lt_wait(qraw + 8 * (c % T::QBUF), (uint32_t)(c / T::QBUF) & 1u, abort_flag, 7)) break;
        if (relu) {
          unsigned char* qt = qrow + c % T::QBUF * T::KTILE;
#pragma unroll
          for (int i = 0; i < PIECES; ++i) {
            uint4* p = reinterpret_cast<uint4*>(qt + piece(i * PARTS + part));
            *p = relu4(*p);
          }
        }
        publish(qfull);
      } else {
        publish(kempty);  // the fence holds back the hand-over until the loads are done: without ReLU nothing else has waited for them
      }
      if (!lt_wait(wempty + wbar, ph ^ 1u, abort_flag, 6)) break;
      const float wt = live ? pow_s[nv - 1 - row] : 0.f;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const int ch = i * PARTS + part;
        uint32_t w[4] = {live ? r[i].x : 0u, live ? r[i].y : 0u, live ? r[i].z : 0u, live ? r[i].w : 0u};  // rows behind the sequence
        float2 x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __fmul2_rn(make_float2(bf16_lo(w[e]), bf16_hi(w[e])), make_float2(wt, wt));
#pragma unroll
        for (int s = 0; s < NT; ++s) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = pack_bf16(x[e].x, x[e].y);
            if (s + 1 < NT) x[e] = __fadd2_rn(x[e], make_float2(-bf16_lo(w[e]), -bf16_hi(w[e])));
          }
          const uint32_t at = T::STACK ? piece(ch + 4 * s) : (uint32_t)(s * T::KTILE) + piece(ch);
          *reinterpret_cast<uint4*>(smem + T::OFF_W + row * 128 + at) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      publish(wfull + wbar);
      unsigned char* vt = vrow + c % T::VBUF * T::VTILE;
      if (!lt_wait(vraw + 8 * (c % T::VBUF), (uint32_t)(c / T::VBUF) & 1u, abort_flag, 8)) break;
      if (!live) {  // rows behind the sequence meet zero weights: they must be finite
#pragma unroll 1
        for (int i = 0; i < PIECES; ++i) *reinterpret_cast<uint4*>(vt + piece(i * PARTS + part)) = make_uint4(0u, 0u, 0u, 0u);
      }
      // An infinity or NaN in v would meet the zero scores of the tokens before it: it is taken out here, and the state and
      // output warps put NaN where it belongs, from its token on.
      uint32_t big = 0u;
      if (look) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
          const uint4 v = *reinterpret_cast<const uint4*>(vt + piece(i * PARTS + part));
          big = __vmaxu2(big, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
        }
      }
      if (live && max(big & 0xffffu, big >> 16) >= 0x7f80u) {
#pragma unroll 1
        for (int k = 0; k < 8 * PIECES; ++k) {
          const int ch = (k >> 3) * PARTS + part;
          unsigned short* p = reinterpret_cast<unsigned short*>(vt + piece(ch)) + (k & 7);
          if ((*p & 0x7fffu) >= 0x7f80u) {
            atomicMin(bad_from + c % T::BADS * D + 8 * ch + (k & 7), row);
            *p = 0;
          }
        }
        bad_flag[c % T::BADS] = 1;
      }
      if (D % 64 != 0 && part == 0) *reinterpret_cast<uint32_t*>(vt + piece(D / 8)) = 0x3f80u;  // the copy put zeros there
      publish(vfull);
    }
  } else {
    // ------------------------------- products -------------------------------------------
    if constexpr (T::WIDE) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp == 8 + LW) {  // the whole warp waits, one elected lane issues
      const uint32_t Wu = sm + T::OFF_W, Vu = sm + T::OFF_V, Ku = sm + T::OFF_K, Qu = sm + T::OFF_Q, Su = sm + T::OFF_S;
      auto wait = [&](uint32_t bb, uint32_t parity, int code) -> bool {
        return lt_wait(bb, parity, abort_flag, code);
      };
      auto qtile = [&](int c) -> uint32_t { return Qu + (uint32_t)(c % T::QBUF * T::KTILE); };
      auto scores = [&](int c, int half) -> bool {  // keys 64 half .. + 63 of chunk c
        const uint32_t ph = (uint32_t)(c & 1);
        if (half == 0 && (!wait(kfull, ph, 17) || !wait(qfull, ph, 11))) return false;
        tcgen05_fence_after();
        if (elect_one()) {
          const uint32_t Qc = qtile(c);
#pragma unroll 1
          for (int k = 0; k < D / 16; ++k)
            umma_bf16(tmem + T::COL_SC + 64 * half, make_smem_desc(Qc + (k >> 2) * LT_BLK) + (uint64_t)(2 * (k & 3)),
                      make_smem_desc(Ku + half * 8192 + (k >> 2) * LT_BLK) + (uint64_t)(2 * (k & 3)), T::ID_SC, k != 0 ? 1u : 0u);
          umma_commit(scready + 8 * half);
          if (half == 1) umma_commit(kempty);
        }
        __syncwarp();
        return true;
      };
      bool ok = !OUT || chunks == 0 || (scores(0, 0) && scores(0, 1));
      for (int c = 0; c < chunks && ok; ++c) {
        const uint32_t ph = (uint32_t)(c & 1);
        const uint64_t vdesc = lt_desc_mn(Vu + (uint32_t)(c % T::VBUF * T::VTILE), LT_BLK);
        if (!wait(wfull, ph, 10) || !wait(wfull + 8, ph, 10) || !wait(vfull, ph, 13) || !wait(dsread, ph ^ 1u, 14)) break;
        tcgen05_fence_after();
        if (elect_one()) {
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
#pragma unroll 1
            for (int s = T::MMAS - 1; s >= 0; --s) {  // smallest term first
              const uint64_t wdesc = lt_desc_mn(Wu + s * T::KTILE, LT_BLK);
#pragma unroll 1
              for (int k = 4 * half; k < 4 * half + 4; ++k)
                umma_bf16(tmem + T::COL_DS, wdesc + (uint64_t)(128 * k), vdesc + (uint64_t)(128 * k), T::ID_DS,
                          (half != 0 || s != T::MMAS - 1 || k != 0) ? 1u : 0u);
            }
            umma_commit(wempty + 8 * half);
          }
          umma_commit(dsready);
          if (!OUT) umma_commit(vempty + 8 * (c % T::VBUF));
        }
        __syncwarp();
        if (!OUT) continue;
        if (!wait(sopready, ph, 15) || !wait(oread, ph ^ 1u, 12)) break;
        tcgen05_fence_after();
        if (elect_one()) {
          const uint32_t Qc = qtile(c);
#pragma unroll 1
          for (int s = T::ST - 1; s >= 0; --s) {  // smallest term first
            const uint64_t sdesc = lt_desc_mn(Su + s * T::VB * T::STATE_BLK, T::STATE_BLK);
#pragma unroll 1
            for (int k = 0; k < D / 16; ++k)
              umma_bf16(tmem + T::COL_O1, make_smem_desc(Qc + (k >> 2) * LT_BLK) + (uint64_t)(2 * (k & 3)), sdesc + (uint64_t)(128 * k),
                        T::ID_O1, (s != T::ST - 1 || k != 0) ? 1u : 0u);
          }
          umma_commit(qempty + 8 * (c % T::QBUF));
          umma_commit(sopread);
        }
        __syncwarp();
        // The decayed scores of a half meet v, then the next chunk's scores take their columns (products run in order) - at
        // once where k and q are there already, else after the other half.
        bool early = false;
#pragma unroll 1
        for (int half = 0; half < 2 && ok; ++half) {
          if (!wait(pready + 8 * half, ph, 16)) { ok = false; break; }
          tcgen05_fence_after();
          if (!T::ALIAS || half == 1) {
            if (elect_one()) {
#pragma unroll 1
              for (int k = T::ALIAS ? 0 : 4 * half; k < 4 * half + 4; ++k) {
                const uint32_t at = tmem + (uint32_t)T::pair_col(k >> 1) + 8u * (k & 1);
                const bool two = T::two_terms(k >> 1);
                if (two) lt_mma_ts(tmem + T::COL_O2, at + 16u, vdesc + (uint64_t)(128 * k), T::ID_O2, k != 0 ? 1u : 0u);
                lt_mma_ts(tmem + T::COL_O2, at, vdesc + (uint64_t)(128 * k), T::ID_O2, k != 0 || two ? 1u : 0u);
              }
              if (half == 1) {
                umma_commit(vempty + 8 * (c % T::VBUF));
                umma_commit(oready);
              }
            }
            __syncwarp();
          }
          if (!T::ALIAS && half == 0 && c + 1 < chunks) {
            early = __all_sync(0xffffffffu, lt_test(kfull, ph ^ 1u) && lt_test(qfull, ph ^ 1u));
            if (early) ok = scores(c + 1, 0);
          }
        }
        if (!T::ALIAS && ok && c + 1 < chunks) ok = (early || scores(c + 1, 0)) && scores(c + 1, 1);
        if (T::ALIAS && ok && c + 1 < chunks) ok = wait(oread, ph, 12) && scores(c + 1, 0) && scores(c + 1, 1);
      }
    } else if (warp == 9 + LW) {  // copies; the warp stays together (a lane that waits alone holds up the others' poll for long)
      const int hk = h / a.group;
      auto copy = [&](uint32_t dst, const CUtensorMap* tm, uint32_t full, int head, int n0) {
        if (!elect_one()) return;
        mbar_expect_tx(full, (uint32_t)T::KTILE);
#pragma unroll
        for (int i = 0; i < T::KB; ++i)
          asm volatile(
              "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
              ::"r"(dst + i * LT_BLK), "l"(tm), "r"(full), "r"(64 * i), "r"(head), "r"(n0), "r"(b)
              : "memory");
      };
      // a tile is free only shortly before it is needed again: what it will take is brought into L2 two chunks ahead
      auto prefetch = [&](const CUtensorMap* tm, int head, int n0) {
        if (!elect_one()) return;
#pragma unroll
        for (int i = 0; i < T::KB; ++i)
          asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global [%0, {%1, %2, %3, %4}];" ::"l"(tm), "r"(64 * i), "r"(head), "r"(n0), "r"(b)
                       : "memory");
      };
      for (int c = 0; c < chunks; ++c) {
        const uint32_t ph = (uint32_t)(c & 1);
        const int n0 = n_begin + c * C;
        for (int ahead = c == 0 ? 1 : 2; ahead <= 2; ++ahead)
          if (c + ahead < chunks) {
            prefetch(&tmK, hk, n0 + ahead * C);
            if (OUT) prefetch(&tmQ, h, n0 + ahead * C);
            prefetch(&tmV, hk, n0 + ahead * C);
          }
        if (!lt_wait(kempty, ph ^ 1u, abort_flag, 17)) break;
        copy(sm + T::OFF_K, &tmK, kraw, hk, n0);
        __syncwarp();
        if (OUT) {
          const int qb = c % T::QBUF;
          if (!lt_wait(qempty + 8 * qb, ((uint32_t)(c / T::QBUF) & 1u) ^ 1u, abort_flag, 18)) break;
          copy(sm + T::OFF_Q + (uint32_t)(qb * T::KTILE), &tmQ, qraw + 8 * qb, h, n0);
        __syncwarp();
        }
        const int vb = c % T::VBUF;
        if (!lt_wait(vempty + 8 * vb, ((uint32_t)(c / T::VBUF) & 1u) ^ 1u, abort_flag, 19)) break;
        copy(sm + T::OFF_V + (uint32_t)(vb * T::VTILE), &tmV, vraw + 8 * vb, hk, n0);
        __syncwarp();
      }
    }
  }

  __syncwarp();
  if (*abort_flag) {  // give products in flight time to end before tensor memory is freed
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000LL) {}
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 0) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)T::TMEM_COLS) : "memory");
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------
struct LdMaps {
  CUtensorMap k, v, q;
};
template <int D, int NT, bool OUT>
static int lt_launch(const LdMaps& m, const LdArgs& a, int nseg, int64_t B, cudaStream_t st) {
  using T = Lt<D, NT, OUT>;
  static OncePerDevice once;
  if (auto first = once.first_time()) {
    cudaError_t e = cudaFuncSetAttribute(la_decay_tc_kernel<D, NT, OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::BYTES);
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(la_decay_tc)");
  }
  la_decay_tc_kernel<D, NT, OUT><<<dim3((unsigned)a.H, (unsigned)nseg, (unsigned)B), T::THREADS, T::BYTES, st>>>(m.k, m.v, m.q, a);
  SANA_LAUNCH_CHECK("la_decay_tc kernel");
  return SANA_OK;
}

// One pass (the state in three terms) when the heads alone fill the GPU; else the sequence is cut: the first launch sums
// every segment exactly, the second computes the outputs with two terms.  128-channel heads always take two (three terms
// of the weighted k do not fit beside the other tiles).
template <int D>
static int lt_run(const LdArgs& a, int64_t B, cudaStream_t st) {
  // (channel, head, token, sample) views of the column blocks; a box is 64 channels of 128 tokens of a head
  LdMaps m;
  const uint32_t box[4] = {64, 1, LT_C, 1};
  auto view = [&](CUtensorMap* tm, const void* p, int64_t ld, int64_t heads) {
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)heads, (uint64_t)a.N, (uint64_t)B};
    const uint64_t strides[3] = {(uint64_t)D * 2, (uint64_t)ld * 2, (uint64_t)ld * 2 * (uint64_t)a.N};
    return make_tmap_tiled(tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, p, dims, strides, box, true);
  };
  int rc = view(&m.k, a.k, a.ldk, a.H / a.group);
  if (!rc) rc = view(&m.v, a.v, a.ldv, a.H / a.group);
  if (!rc) rc = view(&m.q, a.q, a.ldq, a.H);
  if (rc) return rc;
  if constexpr (D < 128) {
    if (a.npart == 0) return lt_launch<D, 3, true>(m, a, 1, B, st);
  }
  rc = lt_launch<D, 3, false>(m, a, a.nseg, B, st);
  if (rc) return rc;
  return lt_launch<D, 2, true>(m, a, a.nseg, B, st);
}

// Cost of a split = waves of CTAs x the time of a segment.  A padded batch is taken to hold lengths spread evenly over
// [0, N]: CTAs behind the end of a sequence leave at once, (segments + 1) / 2 of a sequence's have work, and these fill one
// another's gaps, so the waves are not rounded up.  Its split replaces the first one only where it promises at least 15 %,
// since sequences that all reach N lose by it: 4 x 4096, 16 heads of 64, four segments against two, lengths spread 66-86
// us, one long sequence 64 and all full 121 against 94-109 for any.
LdPlan ld_tc_plan(int64_t B, int64_t N, int64_t H, int64_t D, bool ragged, int* npart) {
  const int64_t units = B * H, slots = (int64_t)sm_count() * (D <= 32 ? 2 : 1), chunks = ceil_div(N, LT_C);
  auto segment = [&](int64_t len, int64_t real) -> int64_t {  // tenths of a chunk
    return real > 1 || D == 128 ? 16 * len + 20 + 2 * real : 12 * len + 10;
  };
  auto spread = [&](int64_t len, int64_t real) -> double {
    const double waves = 0.5 * (double)(units * (real + 1)) / (double)slots;
    return (waves > 1. ? waves : 1.) * (double)segment(len, real);
  };
  int64_t best = -1, best_len = chunks;
  for (int64_t n = 1; n <= chunks && n <= 64; ++n) {
    const int64_t len = ceil_div(chunks, n), real = ceil_div(chunks, len);
    const int64_t cost = ceil_div(units * real, slots) * segment(len, real);
    if (best < 0 || cost < best) best = cost, best_len = len;
  }
  if (ragged && B > 1) {
    double limit = 0.85 * spread(best_len, ceil_div(chunks, best_len));
    for (int64_t n = 1; n <= chunks && n <= 64; ++n) {
      const int64_t len = ceil_div(chunks, n);
      const double cost = spread(len, ceil_div(chunks, len));
      if (cost < limit) limit = cost, best_len = len;
    }
  }
  LdPlan p;
  p.seg_len = (int)(best_len * LT_C);
  p.nseg = (int)ceil_div(N, (int64_t)p.seg_len);
  *npart = (p.nseg > 1 || D == 128) ? p.nseg : 0;
  return p;
}

int launch_decay_tc(LdArgs& a, int64_t B, int64_t D, cudaStream_t st) {
  a.wide_rows = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0 && a.ldo % 16 == 0;
  switch (D) {
    case 16: return lt_run<16>(a, B, st);
    case 32: return lt_run<32>(a, B, st);
    case 48: return lt_run<48>(a, B, st);
    case 64: return lt_run<64>(a, B, st);
    case 80: return lt_run<80>(a, B, st);
    case 96: return lt_run<96>(a, B, st);
    case 112: return lt_run<112>(a, B, st);
    default: return lt_run<128>(a, B, st);
  }
}

}  // namespace sana

extern "C" int sana_la_decay_take_device_status(int* status_out) {
  if (!status_out) return sana::fail(SANA_ERR_INVALID, "sana_la_decay_take_device_status: null pointer");
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, sana::g_ld_status, sizeof(int));
  if (e != cudaSuccess) return sana::cuda_status(e, "cudaMemcpyFromSymbol(g_ld_status)");
  if (v != 0) {
    int zero = 0;
    e = cudaMemcpyToSymbol(sana::g_ld_status, &zero, sizeof(int));
    if (e != cudaSuccess) return sana::cuda_status(e, "cudaMemcpyToSymbol(g_ld_status)");
  }
  *status_out = v;
  return SANA_OK;
}
