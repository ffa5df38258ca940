// Causal linear attention with a decay for each head, over prompts (chunked) and single tokens (recurrent).
//
//   S_t = lambda S_{t-1} + [v_t ; 1] (x) phi(k_t)        S [D+1, D], row D = the decayed key sum, lambda = exp(log_decay[h])
//   o_t = scale * S_t[:D] phi(q_t)                       or, normalised:  S_t[:D] phi(q_t) / (S_t[D] . phi(q_t) + eps)
//
// phi is the identity or ReLU.  Chunked form: with S the state before a chunk of C tokens (t, s count inside it)
//
//   o_t  = lambda^(t+1) S phi(q_t) + sum_{s <= t} lambda^(t-s) (phi(q_t) . phi(k_s)) v_s
//   S'   = lambda^C S + sum_t lambda^(C-1-t) [v_t ; 1] (x) phi(k_t)
//
// Powers of lambda are always taken at the difference of two positions (never lambda^t * lambda^-s, which overflows for
// a strong decay).
//
// bf16, more than 64 tokens: la_decay_tc.cu.  bf16 kernel here: prompts of at most 64 tokens, one chunk, a CTA for one head
// (narrow heads: several), bound by latency - it starts and ends faster than the tensor-memory kernels' pipeline (64 tokens:
// 8 x 70 heads of 32 channels 10 us against 16, 8 x 16 heads of 128 14 against 21; 20 heads of 112 12 against 11).  The
// state lives in the accumulator registers of the warps: warp w owns value channels 16 w .. 16 w + 15 against all key
// channels.  The accumulator fragment of S is, register for register, the B operand of S phi(q) (rows of S are the columns
// of the product), and the transposed fragment of v that multiplies the scores is the A operand of the state update, so the
// state never moves and v is read from shared memory once.
// The state stays within a few 2^-24 of fp32: the weighted v is split into three bf16 terms (8 bits each) before the
// tensor core sees it.  In S phi(q) the state, and before v the scores, enter as two bf16 terms (2^-17): an output of a few
// tokens would feel one rounding of a score as much as its own.  The normaliser is summed in fp32 from the unrounded scores.
// fp32: the chunked form on the CUDA cores.  A sequence is split over CTAs into segments when there are fewer heads than the
// GPU has room for: a first launch computes what each segment adds to the state, and each CTA of the second combines those
// of the segments before its own, in order (nothing depends on the order in which CTAs run).
#include "la_decay.cuh"

namespace sana {

constexpr int LD_C = 64;   // most tokens of the bf16 kernel
constexpr int LD_CF = 32;  // tokens per chunk, fp32

__device__ __forceinline__ void ld_cp16(uint32_t dst, const void* src, bool valid) {
  const int sz = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(sz) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ld_relu4(uint32_t (&r)[4]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = ld_relu2(r[e]);
}

template <int D>
struct Ld {
  static constexpr int WH = D / 16;                        // warps per head: 16 value channels each
  static constexpr int HG = WH >= 3 ? 1 : 4 / WH;          // heads per CTA
  static constexpr int THREADS = 32 * WH * HG;
  static constexpr int ROW = 2 * D + 16;                   // odd number of 16-byte pieces: ldmatrix without conflicts
  static constexpr int TILE = LD_C * ROW;
  static constexpr int PROW = 2 * LD_C + 16;               // scores; the 16 spare bytes hold the four partial row sums
  static constexpr int OFF_P = 3 * TILE;                   // q, k, v | scores | powers | key sum | q . key sum |
  static constexpr int OFF_POW = OFF_P + 2 * LD_C * PROW;  // two bf16 terms of the scores
  static constexpr int OFF_Z = OFF_POW + 4 * (LD_C + 4);
  static constexpr int OFF_QZ = OFF_Z + 4 * D;
  static constexpr int OFF_BAD = OFF_QZ + 4 * LD_C;         // first token whose v is not finite, by channel
  static constexpr int HEAD_BYTES = OFF_BAD + 4 * D;
  static constexpr int BYTES = HG * HEAD_BYTES;
  static_assert(HEAD_BYTES % 16 == 0, "tiles stay 16-byte aligned");
};

template <int D>
__global__ void __launch_bounds__(Ld<D>::THREADS) la_decay_short_kernel(const LdArgs a) {
  using T = Ld<D>;
  constexpr int WH = T::WH, KT = D / 16, C = LD_C;
  extern __shared__ __align__(16) unsigned char smem_all[];
  const int hg = threadIdx.x / (32 * WH), tid = threadIdx.x % (32 * WH), wh = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c2 = 2 * (lane & 3);
  unsigned char* smem = smem_all + hg * T::HEAD_BYTES;
  const uint32_t sm = smem_u32(smem);
  float* pow_s = reinterpret_cast<float*>(smem + T::OFF_POW);
  float* z_s = reinterpret_cast<float*>(smem + T::OFF_Z);
  float* qz_s = reinterpret_cast<float*>(smem + T::OFF_QZ);
  int* bad_s = reinterpret_cast<int*>(smem + T::OFF_BAD);
  const int h = blockIdx.x * T::HG + hg, b = blockIdx.z;
  const bool active = h < a.H;  // inactive head groups of the last CTA only keep the barriers
  const int nv = a.lengths ? min(max(a.lengths[b], 0), a.N) : a.N;
  const float gl = active ? a.log_decay[h] : 0.f;
  const int hk = h / a.group;
  const int64_t row0 = (int64_t)b * a.N;
  const bool relu = a.relu != 0;
  if (active) {
    const __nv_bfloat16* qp = static_cast<const __nv_bfloat16*>(a.q) + row0 * a.ldq + (int64_t)h * D;
    const __nv_bfloat16* kp = static_cast<const __nv_bfloat16*>(a.k) + row0 * a.ldk + (int64_t)hk * D;
    const __nv_bfloat16* vp = static_cast<const __nv_bfloat16*>(a.v) + row0 * a.ldv + (int64_t)hk * D;
    for (int i = tid; i < C * (D / 8); i += 32 * WH) {
      const int r = i / (D / 8), ch = i % (D / 8);
      const bool ok = r < nv;
      const int64_t t = ok ? r : 0;  // a valid address; nothing is read from it
      const uint32_t dst = sm + r * T::ROW + ch * 16;
      ld_cp16(dst, qp + t * a.ldq + 8 * ch, ok);
      ld_cp16(dst + T::TILE, kp + t * a.ldk + 8 * ch, ok);
      ld_cp16(dst + 2 * T::TILE, vp + t * a.ldv + 8 * ch, ok);
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  for (int i = tid; i <= C; i += 32 * WH) pow_s[i] = ld_power(gl, i);
  for (int i = tid; i < D; i += 32 * WH) bad_s[i] = C;

  // state: rows 16 wh + g and + 8 (value channels), columns 8 n + c2, + 1 (key channels); zacc: rows 0..2 hold the three
  // terms of the key sum of columns 16 wh + 8 n + c2, + 1
  float S[2 * KT][4], zacc[2][4];
#pragma unroll
  for (int n = 0; n < 2 * KT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) S[n][e] = 0.f;
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) zacc[n][e] = 0.f;
  const int64_t per = (int64_t)(D + 1) * D;
  if (a.prior && active) {
    const float* src = a.prior + ((int64_t)b * a.H + h) * per;
    const float* r = src + (int64_t)(16 * wh + g) * D + c2;
#pragma unroll
    for (int n = 0; n < 2 * KT; ++n) {
      const float2 u = __ldg(reinterpret_cast<const float2*>(r + 8 * n));
      const float2 w = __ldg(reinterpret_cast<const float2*>(r + 8 * D + 8 * n));
      S[n][0] = u.x, S[n][1] = u.y, S[n][2] = w.x, S[n][3] = w.y;
    }
    if (g == 0) {
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const float2 u = __ldg(reinterpret_cast<const float2*>(src + (int64_t)D * D + 16 * wh + 8 * n + c2));
        zacc[n][0] = u.x, zacc[n][1] = u.y;
      }
    }
  }
  {  // the key sum into shared memory: the three terms are rows 0, 1, 2 = lanes 4 g
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float z = zacc[n][e];
        z += __shfl_down_sync(0xffffffffu, zacc[n][e], 4) + __shfl_down_sync(0xffffffffu, zacc[n][e], 8);
        if (g == 0) z_s[16 * wh + 8 * n + c2 + e] = z;
      }
  }

  // ldmatrix addresses inside a tile: 16 rows x 16 columns as four 8 x 8 matrices
  const uint32_t off_rows = (lane & 15) * T::ROW + (lane >> 4) * 16;                       // (rows 0-7, 8-15) x (columns 0-7, 8-15)
  const uint32_t off_cols = ((lane & 7) + (lane >> 4) * 8) * T::ROW + ((lane >> 3) & 1) * 16;  // columns first
  const uint32_t Qs = sm, Ks = Qs + T::TILE, Vs = Ks + T::TILE, Ps = sm + T::OFF_P;
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  // An infinity or NaN in v would meet the zero scores of the tokens before it: it is taken out, and NaN put where it belongs.
  bool odd = false;
  if (active) {
    for (int i = tid; i < C * (D / 8); i += 32 * WH) {  // the pieces this thread has loaded
      const int r = i / (D / 8), ch = i % (D / 8);
      unsigned short* p = reinterpret_cast<unsigned short*>(smem + 2 * T::TILE + r * T::ROW + ch * 16);
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
      odd |= max(m & 0xffffu, m >> 16) >= 0x7f80u;
    }
  }
  odd = __syncthreads_or(odd);  // the tiles are there
  if (odd) {
    if (active)
      for (int i = tid; i < C * D; i += 32 * WH) {
        const int r = i / D, ch = i % D;
        unsigned short* p = reinterpret_cast<unsigned short*>(smem + 2 * T::TILE + r * T::ROW) + ch;
        if ((*p & 0x7fffu) >= 0x7f80u) {
          atomicMin(bad_s + ch, r);
          *p = 0;
        }
      }
    __syncthreads();
  }
  if (active) {
    // scores of the 16 x 16 blocks on and below the diagonal, dealt to the warps in turn
    int id = 0;
    for (int mi = 0; mi * 16 < nv; ++mi) {
      for (int ni = 0; ni <= mi; ++ni, ++id) {
        if (id % WH != wh) continue;
        float p[2][4] = {};
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          uint32_t qa[4], kb[4];
          ldsm_x4(qa, Qs + mi * 16 * T::ROW + off_rows + kt * 32);
          ldsm_x4(kb, Ks + ni * 16 * T::ROW + off_cols + kt * 32);
          if (relu) ld_relu4(qa), ld_relu4(kb);
          mma_bf16_16816(p[0], qa[0], qa[1], qa[2], qa[3], kb[0], kb[1]);
          mma_bf16_16816(p[1], qa[0], qa[1], qa[2], qa[3], kb[2], kb[3]);
        }
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = 16 * (mi - ni) + g + 8 * (e >> 1) - (8 * n + c2 + (e & 1));  // t - s
            p[n][e] = d >= 0 ? p[n][e] * pow_s[d] : 0.f;
            sum[e >> 1] += p[n][e];
          }
        unsigned char* pr = smem + T::OFF_P + (16 * mi + g) * T::PROW;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          unsigned char* at = pr + 2 * (16 * ni + 8 * n + c2);
          *reinterpret_cast<uint32_t*>(at) = ld_split(p[n][0], p[n][1]);
          *reinterpret_cast<uint32_t*>(at + 8 * T::PROW) = ld_split(p[n][2], p[n][3]);
          *reinterpret_cast<uint32_t*>(at + C * T::PROW) = pack_bf16(p[n][0], p[n][1]);
          *reinterpret_cast<uint32_t*>(at + (C + 8) * T::PROW) = pack_bf16(p[n][2], p[n][3]);
        }
        if (a.normalise) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 1);
            sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], 2);
            if (c2 == 0) *reinterpret_cast<float*>(pr + 8 * e * T::PROW + 2 * C + 4 * ni) = sum[e];
          }
        }
      }
    }
    if (a.normalise) {  // q . key sum, the key sum as two bf16 terms in columns 0 and 1 of the B operand
      for (int mi = wh; mi * 16 < nv; mi += WH) {
        float d[4] = {};
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          uint32_t qa[4];
          ldsm_x4(qa, Qs + mi * 16 * T::ROW + off_rows + kt * 32);
          if (relu) ld_relu4(qa);
          uint32_t zb[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float2 z = *reinterpret_cast<const float2*>(z_s + 16 * kt + 8 * e + c2);
            const uint32_t hi = ld_split(z.x, z.y);
            zb[e] = g == 0 ? hi : g == 1 ? pack_bf16(z.x, z.y) : 0u;
          }
          mma_bf16_16816(d, qa[0], qa[1], qa[2], qa[3], zb[0], zb[1]);
        }
        if (c2 == 0) {
          qz_s[16 * mi + g] = d[0] + d[1];
          qz_s[16 * mi + g + 8] = d[2] + d[3];
        }
      }
    }
  }
  __syncthreads();  // scores and normalisers are there
  if (!active) return;
  uint32_t vf[4][4];  // v of the chunk, this warp's 16 channels: [token tile][(s 0-7, ch 0-7), (s 8-15, 0-7), (0-7, 8-15), (8-15, 8-15)]
#pragma unroll
  for (int kt = 0; kt < 4; ++kt) ldsm_x4_t(vf[kt], Vs + kt * 16 * T::ROW + off_rows + wh * 32);
  float o[4][2][4] = {};
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {  // S phi(q): key channels 16 kt ..
    uint32_t hi[2][2], lo[2][2];     // [rows of S 0-7, 8-15 = output column tile][k half]
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = S[2 * kt + e][2 * r], y = S[2 * kt + e][2 * r + 1];
        hi[r][e] = ld_split(x, y);
        lo[r][e] = pack_bf16(x, y);
      }
#pragma unroll
    for (int mi = 0; mi < 4; ++mi) {
      uint32_t qa[4];
      ldsm_x4(qa, Qs + mi * 16 * T::ROW + off_rows + kt * 32);
      if (relu) ld_relu4(qa);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        mma_bf16_16816(o[mi][r], qa[0], qa[1], qa[2], qa[3], hi[r][0], hi[r][1]);
        mma_bf16_16816(o[mi][r], qa[0], qa[1], qa[2], qa[3], lo[r][0], lo[r][1]);
      }
    }
  }
#pragma unroll
  for (int mi = 0; mi < 4; ++mi) {
    if (16 * mi >= nv) break;
    const float f0 = pow_s[16 * mi + g + 1], f1 = pow_s[16 * mi + g + 9];
#pragma unroll
    for (int r = 0; r < 2; ++r) o[mi][r][0] *= f0, o[mi][r][1] *= f0, o[mi][r][2] *= f1, o[mi][r][3] *= f1;
#pragma unroll
    for (int kt = 0; kt <= mi; ++kt) {
      uint32_t pa[4];
#pragma unroll
      for (int s = 1; s >= 0; --s) {  // the second terms first
        ldsm_x4(pa, Ps + (s * C + 16 * mi + (lane & 15)) * T::PROW + (lane >> 4) * 16 + kt * 32);
        mma_bf16_16816(o[mi][0], pa[0], pa[1], pa[2], pa[3], vf[kt][0], vf[kt][1]);
        mma_bf16_16816(o[mi][1], pa[0], pa[1], pa[2], pa[3], vf[kt][2], vf[kt][3]);
      }
    }
    float m0 = a.scale, m1 = a.scale;
    if (a.normalise) {
      const unsigned char* pr = smem + T::OFF_P + (16 * mi + g) * T::PROW + 2 * C;
      float d0 = f0 * qz_s[16 * mi + g], d1 = f1 * qz_s[16 * mi + g + 8];
#pragma unroll
      for (int ni = 0; ni <= mi; ++ni) {
        d0 += *reinterpret_cast<const float*>(pr + 4 * ni);
        d1 += *reinterpret_cast<const float*>(pr + 8 * T::PROW + 4 * ni);
      }
      m0 = 1.f / (d0 + a.eps);
      m1 = 1.f / (d1 + a.eps);
    }
    if (odd) {
      const float nan = __uint_as_float(0x7fffffffu);
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (16 * mi + g + 8 * (e >> 1) >= bad_s[16 * wh + 8 * r + c2 + (e & 1)]) o[mi][r][e] = nan;
    }
    // the four lanes of a row group swap so that each holds 16 bytes of one row: lane 0 / 1 row g, channels 0-7 / 8-15,
    // lane 2 / 3 the same of row g + 8
    uint32_t w[4] = {pack_bf16(o[mi][0][0] * m0, o[mi][0][1] * m0), pack_bf16(o[mi][1][0] * m0, o[mi][1][1] * m0),
                     pack_bf16(o[mi][0][2] * m1, o[mi][0][3] * m1), pack_bf16(o[mi][1][2] * m1, o[mi][1][3] * m1)};
    const int c = lane & 3;
#pragma unroll
    for (int s = 1; s < 4; s <<= 1) {  // transpose by exchanging with lane c ^ s
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i & s) continue;
        const uint32_t give = (c & s) ? w[i] : w[i | s];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, give, s);
        if (c & s) w[i] = got; else w[i | s] = got;
      }
    }
    const int t = 16 * mi + g + 8 * (c >> 1);
    if (t < nv)
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + (row0 + t) * a.ldo + (int64_t)h * D + 16 * wh +
                                8 * (c & 1)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  // state update: S = lambda^nv S + (weighted v)^T k.  The tensor core truncates its fp32 sums, so a chunk is summed on
  // its own, smallest terms first, and joined to the state by one rounded multiply-add.
  const float whole = pow_s[nv];
  uint32_t va[4][3][4], wa[4][2];  // three terms of the weighted v (A operand); terms of the weights in rows 0..2
#pragma unroll
  for (int kt = 0; kt < 4; ++kt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // tokens 16 kt + 8 e + c2, + 1
      const int left = nv - 1 - (16 * kt + 8 * e + c2);
      float w0 = left >= 0 ? pow_s[left] : 0.f, w1 = left >= 1 ? pow_s[left - 1] : 0.f;
#pragma unroll
      for (int r = 0; r < 2; ++r) {  // channels 0-7, 8-15: fragment register vf[2 r + e], A register 2 e + r
        float x = bf16_lo(vf[kt][2 * r + e]) * w0, y = bf16_hi(vf[kt][2 * r + e]) * w1;
#pragma unroll
        for (int s = 0; s < 3; ++s) va[kt][s][2 * e + r] = ld_split(x, y);
      }
      const uint32_t t0 = ld_split(w0, w1), t1 = ld_split(w0, w1), t2 = ld_split(w0, w1);
      wa[kt][e] = g == 0 ? t0 : g == 1 ? t1 : g == 2 ? t2 : 0u;
    }
#pragma unroll
  for (int n = 0; n < KT; ++n) {
    uint32_t kb[4][4];  // k[tokens][16 n ..] as the B operand of two column tiles
    float d[2][4] = {};
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      ldsm_x4_t(kb[kt], Ks + kt * 16 * T::ROW + off_rows + n * 32);
      if (relu) ld_relu4(kb[kt]);
    }
#pragma unroll
    for (int s = 2; s >= 0; --s)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        mma_bf16_16816(d[0], va[kt][s][0], va[kt][s][1], va[kt][s][2], va[kt][s][3], kb[kt][0], kb[kt][1]);
        mma_bf16_16816(d[1], va[kt][s][0], va[kt][s][1], va[kt][s][2], va[kt][s][3], kb[kt][2], kb[kt][3]);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) S[2 * n + r][e] = fmaf(whole, S[2 * n + r][e], d[r][e]);
    if (n == wh) {
      float z[2][4] = {};
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        mma_bf16_16816(z[0], wa[kt][0], 0u, wa[kt][1], 0u, kb[kt][0], kb[kt][1]);
        mma_bf16_16816(z[1], wa[kt][0], 0u, wa[kt][1], 0u, kb[kt][2], kb[kt][3]);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int e = 0; e < 2; ++e) zacc[r][e] = fmaf(whole, zacc[r][e], z[r][e]);
    }
  }
  if (odd) {
#pragma unroll
    for (int n = 0; n < 2 * KT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (bad_s[16 * wh + g + 8 * (e >> 1)] < C) S[n][e] = __uint_as_float(0x7fffffffu);
  }
  float* dst = a.state + ((int64_t)b * a.H + h) * per;
  float* r = dst + (int64_t)(16 * wh + g) * D + c2;
#pragma unroll
  for (int n = 0; n < 2 * KT; ++n) {
    *reinterpret_cast<float2*>(r + 8 * n) = make_float2(S[n][0], S[n][1]);
    *reinterpret_cast<float2*>(r + 8 * D + 8 * n) = make_float2(S[n][2], S[n][3]);
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    float z[2];
#pragma unroll
    for (int e = 0; e < 2; ++e)
      z[e] = zacc[n][e] + __shfl_down_sync(0xffffffffu, zacc[n][e], 4) + __shfl_down_sync(0xffffffffu, zacc[n][e], 8);
    if (g == 0) *reinterpret_cast<float2*>(dst + (int64_t)D * D + 16 * wh + 8 * n + c2) = make_float2(z[0], z[1]);
  }
  for (int i = tid; i < (a.N - nv) * (D / 8); i += 32 * WH) {  // rows past the sequence are zeros
    const int t = nv + i / (D / 8), ch = i % (D / 8);
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + (row0 + t) * a.ldo + (int64_t)h * D + 8 * ch) = make_uint4(0u, 0u, 0u, 0u);
  }
}

// ---- fp32: the same chunked form on the CUDA cores, state in shared memory ------------------------------------------
// Bound by the fp32 pipes and the barriers between a chunk's four steps: 2 x 1001 tokens, 8 heads of 32 channels 48-55 us.
// For tests and small models; chunks of 32 keep the work of the triangle (quadratic in the chunk) below that of the state.
template <int D>
struct LdF {
  static constexpr int ROW = D + 4;
  static constexpr int TILE = LD_CF * ROW;
  static constexpr int FLOATS = 3 * TILE + (D + 1) * ROW + LD_CF * (LD_CF + 1) + (LD_CF + 4);
};

template <int D, bool OUT>
__global__ void __launch_bounds__(256) la_decay_f32_kernel(const LdArgs a) {
  using T = LdF<D>;
  constexpr int C = LD_CF, ROW = T::ROW, E = D / 16;
  extern __shared__ __align__(16) float fsm[];
  float *qs = fsm, *ks = qs + T::TILE, *vs = ks + T::TILE, *ss = vs + T::TILE;  // ss [D+1][ROW]
  float *ps = ss + (D + 1) * ROW, *pw = ps + C * (C + 1);
  const int tid = threadIdx.x;
  const int h = blockIdx.x, seg = blockIdx.y, b = blockIdx.z;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.N) : a.N;
  const int seg_begin = seg * a.seg_len, seg_end = min(a.N, seg_begin + a.seg_len);
  const int n_begin = min(seg_begin, len), n_end = min(seg_end, len);
  const float gl = a.log_decay[h];
  const int64_t row0 = (int64_t)b * a.N;
  const float* qp = static_cast<const float*>(a.q) + row0 * a.ldq + (int64_t)h * D;
  const float* kp = static_cast<const float*>(a.k) + row0 * a.ldk + (int64_t)(h / a.group) * D;
  const float* vp = static_cast<const float*>(a.v) + row0 * a.ldv + (int64_t)(h / a.group) * D;
  const int64_t per = (int64_t)(D + 1) * D;
  for (int i = tid; i <= C; i += 256) pw[i] = ld_power(gl, i);
  for (int i = tid; i < (D + 1) * D; i += 256) {
    float x = 0.f;
    if (OUT) {
      if (a.prior) x = ld_power(gl, n_begin) * a.prior[((int64_t)b * a.H + h) * per + i];
      for (int r = 0; r < seg; ++r) {
        const int end = min((r + 1) * a.seg_len, len);
        if (end == min(r * a.seg_len, len)) break;
        x = fmaf(ld_power(gl, n_begin - end), a.partial[(((int64_t)b * a.npart + r) * a.H + h) * per + i], x);
      }
    }
    ss[(i / D) * ROW + i % D] = x;
  }
  for (int n0 = n_begin; n0 < n_end; n0 += C) {
    const int nv = min(C, n_end - n0);
    __syncthreads();
    for (int i = tid; i < C * (D / 4); i += 256) {
      const int r = i / (D / 4), ch = 4 * (i % (D / 4));
      float4 q = make_float4(0.f, 0.f, 0.f, 0.f), k = q, v = q;
      if (r < nv) {
        if (OUT) q = __ldg(reinterpret_cast<const float4*>(qp + (int64_t)(n0 + r) * a.ldq + ch));
        k = __ldg(reinterpret_cast<const float4*>(kp + (int64_t)(n0 + r) * a.ldk + ch));
        v = __ldg(reinterpret_cast<const float4*>(vp + (int64_t)(n0 + r) * a.ldv + ch));
      }
      if (a.relu) {  // a comparison, not fmaxf: a NaN stays one
        q.x = q.x < 0.f ? 0.f : q.x, q.y = q.y < 0.f ? 0.f : q.y, q.z = q.z < 0.f ? 0.f : q.z, q.w = q.w < 0.f ? 0.f : q.w;
        k.x = k.x < 0.f ? 0.f : k.x, k.y = k.y < 0.f ? 0.f : k.y, k.z = k.z < 0.f ? 0.f : k.z, k.w = k.w < 0.f ? 0.f : k.w;
      }
      *reinterpret_cast<float4*>(qs + r * ROW + ch) = q;
      *reinterpret_cast<float4*>(ks + r * ROW + ch) = k;
      *reinterpret_cast<float4*>(vs + r * ROW + ch) = v;
    }
    __syncthreads();
    if (OUT) {
      const int t = tid >> 3, sub = tid & 7;  // 32 tokens x 8 lanes
      float rs = 0.f;
#pragma unroll
      for (int e = 0; e < C / 8; ++e) {
        const int s = sub + 8 * e;
        float x = 0.f;
        if (s <= t) {
#pragma unroll 4
          for (int j = 0; j < D; j += 4) {
            const float4 u = *reinterpret_cast<const float4*>(qs + t * ROW + j), w = *reinterpret_cast<const float4*>(ks + s * ROW + j);
            x = fmaf(u.x, w.x, fmaf(u.y, w.y, fmaf(u.z, w.z, fmaf(u.w, w.w, x))));
          }
          x *= pw[t - s];
        }
        ps[t * (C + 1) + s] = x;
        rs += x;
      }
      float qz = 0.f;
      for (int j = sub; j < D; j += 8) qz = fmaf(qs[t * ROW + j], ss[D * ROW + j], qz);
      float dsum = fmaf(pw[t + 1], qz, rs);
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) dsum += __shfl_xor_sync(0xffffffffu, dsum, o);
      const float m = a.normalise ? 1.f / (dsum + a.eps) : a.scale;
      __syncwarp();  // a token's eight lanes are in one warp
      float* orow = static_cast<float*>(a.out) + (row0 + n0 + t) * a.ldo + (int64_t)h * D;
#pragma unroll 2
      for (int i = sub; i < D; i += 8) {
        float x = 0.f, y = 0.f;
#pragma unroll 4
        for (int j = 0; j < D; j += 4) {
          const float4 u = *reinterpret_cast<const float4*>(qs + t * ROW + j), w = *reinterpret_cast<const float4*>(ss + i * ROW + j);
          x = fmaf(u.x, w.x, fmaf(u.y, w.y, fmaf(u.z, w.z, fmaf(u.w, w.w, x))));
        }
        for (int s = 0; s <= t; ++s) y = fmaf(ps[t * (C + 1) + s], vs[s * ROW + i], y);
        if (t < nv) orow[i] = fmaf(pw[t + 1], x, y) * m;
      }
    }
    __syncthreads();
    {
      const int ti = tid >> 4, tj = tid & 15;
      float acc[E][E] = {};
      float zc = 0.f;
      for (int s = 0; s < nv; ++s) {
        const float w = pw[nv - 1 - s];
        float vv[E], kk[E];
#pragma unroll
        for (int e = 0; e < E; ++e) vv[e] = w * vs[s * ROW + ti + 16 * e], kk[e] = ks[s * ROW + tj + 16 * e];
#pragma unroll
        for (int i = 0; i < E; ++i)
#pragma unroll
          for (int j = 0; j < E; ++j) acc[i][j] = fmaf(vv[i], kk[j], acc[i][j]);
        if (tid < D) zc = fmaf(w, ks[s * ROW + tid], zc);
      }
      const float whole = pw[nv];
#pragma unroll
      for (int i = 0; i < E; ++i)
#pragma unroll
        for (int j = 0; j < E; ++j) {
          float* p = ss + (ti + 16 * i) * ROW + tj + 16 * j;
          *p = fmaf(whole, *p, acc[i][j]);
        }
      if (tid < D) ss[D * ROW + tid] = fmaf(whole, ss[D * ROW + tid], zc);
    }
  }
  __syncthreads();
  if (!OUT || seg == a.nseg - 1) {
    float* dst = OUT ? a.state + ((int64_t)b * a.H + h) * per : a.partial + (((int64_t)b * a.npart + seg) * a.H + h) * per;
    for (int i = tid; i < (D + 1) * D; i += 256) dst[i] = ss[(i / D) * ROW + i % D];
  }
  if (OUT) {
    const int z0 = max(seg_begin, n_end);
    for (int64_t i = tid; i < (int64_t)max(0, seg_end - z0) * D; i += 256)
      static_cast<float*>(a.out)[(row0 + z0 + i / D) * a.ldo + (int64_t)h * D + i % D] = 0.f;
  }
}

// ---- one token -----------------------------------------------------------------------------------------------------
// A CTA holds the state of one head of one sequence: reads it once, adds the token, writes it back and multiplies it
// with q on the way.  Bound by the state's bytes (8 (D+1) D per head against 4 D^2 operations): 256 sequences of 16 heads of 128
// channels (a state of 270 MB, read and written) 83 us, 6.5 TB/s, the copy rate.  GP lanes share a row; all rows of a thread
// are in flight at once, q, k and v with them (loaded behind the test for repeated slots they cost 12 us).
struct LdStepArgs {
  const void *q, *k, *v;
  int64_t ldq, ldk, ldv;
  const float* log_decay;
  float* state;
  const int* slots;
  void* out;
  int64_t ldo;
  int H, group, pool;
  float scale, eps;
  int relu, normalise;
};

// About eight float4 of the state per thread, so that an SM's CTAs have some 130 KB of it in flight: with 256 threads for
// every width, 256 sequences of 20 heads of 112 took 96 us instead of 83, of 70 heads of 32 channels 45 instead of 25.
constexpr int ld_step_threads(int D) { return D >= 80 ? 512 : D >= 64 ? 256 : D >= 48 ? 128 : 64; }
template <int D, typename T>
__global__ void __launch_bounds__(ld_step_threads(D)) la_decay_step_kernel(const LdStepArgs a) {
  constexpr int V = D / 4;                                                 // float4 pieces of a row
  constexpr int GP = V <= 4 ? 4 : V <= 8 ? 8 : V <= 16 ? 16 : 32;          // lanes per row
  constexpr int RPI = ld_step_threads(D) / GP;                                            // rows per pass of the CTA
  constexpr int PASSES = (D + 1 + RPI - 1) / RPI;
  __shared__ float o_s[D + 1], v_s[D + 1];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int slot = a.slots ? a.slots[b] : b;
  T* out = static_cast<T*>(a.out) + (int64_t)b * a.ldo + (int64_t)h * D;
  if (slot < 0 || slot >= a.pool) {  // -1: a row without a sequence, zeros; anything else is not a slot: NaN
    if (tid < D) out[tid] = from_f32<T>(slot == -1 ? 0.f : __uint_as_float(0x7fffffffu));
    return;
  }
  const int l = tid % GP, r0 = tid / GP;
  const bool in = l < V;
  float* S = a.state + ((int64_t)slot * a.H + h) * (int64_t)((D + 1) * D) + 4 * l;
  float4 s[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int r = r0 + p * RPI;
    s[p] = in && r <= D ? *reinterpret_cast<const float4*>(S + (int64_t)r * D) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // q, k and v are under way with the state
  const float lam = expf(a.log_decay[h]);
  const int hk = h / a.group;
  const T* qp = static_cast<const T*>(a.q) + (int64_t)b * a.ldq + (int64_t)h * D;
  const T* kp = static_cast<const T*>(a.k) + (int64_t)b * a.ldk + (int64_t)hk * D;
  const T* vp = static_cast<const T*>(a.v) + (int64_t)b * a.ldv + (int64_t)hk * D;
  float q[4], k[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    q[e] = in ? to_f32(qp[4 * l + e]) : 0.f;
    k[e] = in ? to_f32(kp[4 * l + e]) : 0.f;
    if (a.relu) q[e] = q[e] < 0.f ? 0.f : q[e], k[e] = k[e] < 0.f ? 0.f : k[e];
  }
  if (tid <= D) v_s[tid] = tid < D ? to_f32(vp[tid]) : 1.f;
  // a slot that an earlier row of the batch already names would be updated by two CTAs at once: such a row is not a
  // step of its own, its output is NaN and the state takes the first row's token only
  bool twice = false;
  if (a.slots)
    for (int i = tid; i < b; i += ld_step_threads(D)) twice |= a.slots[i] == slot;
  if (__syncthreads_or(twice)) {
    if (tid < D) out[tid] = from_f32<T>(__uint_as_float(0x7fffffffu));
    return;
  }
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int r = r0 + p * RPI;
    const float v = v_s[r <= D ? r : D];
    float4 n;
    n.x = fmaf(v, k[0], lam * s[p].x);
    n.y = fmaf(v, k[1], lam * s[p].y);
    n.z = fmaf(v, k[2], lam * s[p].z);
    n.w = fmaf(v, k[3], lam * s[p].w);
    if (in && r <= D) *reinterpret_cast<float4*>(S + (int64_t)r * D) = n;
    float x = fmaf(q[0], n.x, fmaf(q[1], n.y, fmaf(q[2], n.z, q[3] * n.w)));
#pragma unroll
    for (int o = GP / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (l == 0 && r <= D) o_s[r] = x;
  }
  __syncthreads();
  if (tid < D) out[tid] = from_f32<T>(a.normalise ? o_s[tid] / (o_s[D] + a.eps) : o_s[tid] * a.scale);
}

// ---- host ----------------------------------------------------------------------------------------------------------
// CTAs of the fp32 kernel resident at once on the current device; also raises its shared-memory limit there, once.
template <int D>
static int64_t ld_slots() {
  static int64_t known[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
  if (known[dev] > 0) return known[dev];
  cudaFuncSetAttribute(la_decay_f32_kernel<D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, LdF<D>::FLOATS * 4);
  cudaFuncSetAttribute(la_decay_f32_kernel<D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, LdF<D>::FLOATS * 4);
  return known[dev] = resident_ctas(la_decay_f32_kernel<D, true>, 256, LdF<D>::FLOATS * 4);
}

constexpr int64_t LD_TC_TOKENS = LD_C + 1;  // shortest sequences the tcgen05 kernels take

// Token segments and their number; npart = segments whose sums go through the workspace.  fp32: a sequence is cut only when
// the heads alone leave the GPU partly empty, since every cut re-reads k and v.  Cost of a choice = waves x (tokens of a
// segment, plus half as many again for the first launch, plus about two chunks for reading the states before it).
template <int D>
static void ld_plan(int64_t B, int64_t N, int64_t H, int dtype, bool ragged, int* seg_len, int* nseg, int* npart) {
  if (dtype == SANA_BF16) {
    LdPlan p = {LD_C, 1};
    *npart = 0;
    if (N >= LD_TC_TOKENS) p = ld_tc_plan(B, N, H, D, ragged, npart);
    *seg_len = p.seg_len, *nseg = p.nseg;
    return;
  }
  const int64_t units = B * H, slots = ld_slots<D>(), chunks = ceil_div(N, LD_CF);
  int64_t best = -1, best_len = chunks;
  for (int64_t n = 1; n <= chunks && n <= 64; ++n) {
    const int64_t len = ceil_div(chunks, n), real = ceil_div(chunks, len);
    int64_t cost = ceil_div(units * real, slots) * 2 * len;
    if (real > 1) cost += ceil_div(units * (real - 1), slots) * len + 4 + real;
    if (best < 0 || cost < best) best = cost, best_len = len;
  }
  *seg_len = (int)(best_len * LD_CF);
  *nseg = (int)ceil_div(N, (int64_t)*seg_len);
  *npart = *nseg - 1;
}

template <int D>
static int launch_decay(LdArgs& a, int64_t B, int dtype, int64_t workspace_bytes, cudaStream_t st) {
  ld_plan<D>(B, a.N, a.H, dtype, a.lengths != nullptr, &a.seg_len, &a.nseg, &a.npart);
  SANA_REQUIRE(workspace_bytes >= (int64_t)4 * B * a.npart * a.H * (D + 1) * D, "sana_la_decay: workspace too small");
  if (dtype == SANA_BF16) {
    if (a.N >= LD_TC_TOKENS) return launch_decay_tc(a, B, D, st);
    static OncePerDevice once;
    if (auto first = once.first_time()) {
      cudaError_t e = cudaFuncSetAttribute(la_decay_short_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Ld<D>::BYTES);
      if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(la_decay_short)");
    }
    la_decay_short_kernel<D><<<dim3((unsigned)ceil_div(a.H, Ld<D>::HG), 1, (unsigned)B), Ld<D>::THREADS, Ld<D>::BYTES, st>>>(a);
  } else {
    const dim3 grid((unsigned)a.H, (unsigned)a.nseg, (unsigned)B);
    if (a.nseg > 1) {
      la_decay_f32_kernel<D, false><<<dim3(grid.x, a.nseg - 1, grid.z), 256, LdF<D>::FLOATS * 4, st>>>(a);
      SANA_LAUNCH_CHECK("la_decay segment kernel");
    }
    la_decay_f32_kernel<D, true><<<grid, 256, LdF<D>::FLOATS * 4, st>>>(a);
  }
  SANA_LAUNCH_CHECK("la_decay kernel");
  return SANA_OK;
}

template <int D>
static int launch_decay_step(const LdStepArgs& a, int64_t B, int dtype, cudaStream_t st) {
  const dim3 grid((unsigned)a.H, (unsigned)B);
  if (dtype == SANA_BF16) la_decay_step_kernel<D, __nv_bfloat16><<<grid, ld_step_threads(D), 0, st>>>(a);
  else la_decay_step_kernel<D, float><<<grid, ld_step_threads(D), 0, st>>>(a);
  SANA_LAUNCH_CHECK("la_decay_step kernel");
  return SANA_OK;
}

#define LD_DISPATCH(D, CALL)                \
  switch (D) {                              \
    case 16: { constexpr int HD = 16; CALL; } break;   \
    case 32: { constexpr int HD = 32; CALL; } break;   \
    case 48: { constexpr int HD = 48; CALL; } break;   \
    case 64: { constexpr int HD = 64; CALL; } break;   \
    case 80: { constexpr int HD = 80; CALL; } break;   \
    case 96: { constexpr int HD = 96; CALL; } break;   \
    case 112: { constexpr int HD = 112; CALL; } break; \
    case 128: { constexpr int HD = 128; CALL; } break; \
  }

static bool ld_head_dim(int64_t D) { return D >= 16 && D <= 128 && D % 16 == 0; }

static int ld_check(const char* who, int64_t ldq, int64_t ldk, int64_t ldv, int64_t ldo, int64_t H, int64_t Hk, int64_t D, int dtype,
                    const void* q, const void* k, const void* v, const void* out, int relu, float eps) {
  SANA_REQUIRE(ld_head_dim(D), "%s: head dimension %lld is not a multiple of 16 in [16, 128]", who, (long long)D);
  SANA_REQUIRE(dtype == SANA_BF16 || dtype == SANA_F32, "%s: unknown dtype %d", who, dtype);
  SANA_REQUIRE(H > 0 && Hk > 0 && H % Hk == 0 && H <= 65535, "%s: H must be a multiple of the key/value heads, at most 65535", who);
  const int64_t unit = dtype == SANA_BF16 ? 8 : 4;
  SANA_REQUIRE(ldq >= H * D && ldo >= H * D && ldk >= Hk * D && ldv >= Hk * D, "%s: row stride shorter than a row", who);
  SANA_REQUIRE(ldq % unit == 0 && ldk % unit == 0 && ldv % unit == 0 && ldo % unit == 0 && aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out),
               "%s: rows must be 16-byte aligned", who);
  SANA_REQUIRE(!(eps >= 0.f) || relu, "%s: the normalised form needs the ReLU features", who);
  return SANA_OK;
}

}  // namespace sana

using namespace sana;

extern "C" int64_t sana_la_decay_plan(int64_t B, int64_t N, int64_t H, int64_t D, int dtype, int ragged, int* launches) {
  if (B <= 0 || N <= 0 || N >= ((int64_t)1 << 30) || H <= 0 || !ld_head_dim(D) || (dtype != SANA_BF16 && dtype != SANA_F32)) return -1;
  int len = 0, nseg = 1, npart = 0;
  LD_DISPATCH(D, (ld_plan<HD>(B, N, H, dtype, ragged != 0, &len, &nseg, &npart)));
  if (launches) *launches = npart > 0 ? 2 : 1;  // segments are summed by a launch of their own
  return (int64_t)4 * B * npart * H * (D + 1) * D;
}

extern "C" int64_t sana_la_decay_workspace_bytes(int64_t B, int64_t N, int64_t H, int64_t D, int dtype) {
  const int64_t even = sana_la_decay_plan(B, N, H, D, dtype, 0, nullptr), ragged = sana_la_decay_plan(B, N, H, D, dtype, 1, nullptr);
  return even > ragged ? even : ragged;
}

extern "C" int sana_la_decay(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, const float* log_decay,
                             const float* prior, const int32_t* lengths, float* state, void* out, int64_t ldo, void* workspace,
                             int64_t workspace_bytes, int64_t B, int64_t N, int64_t H, int64_t Hk, int64_t D, float scale,
                             int relu, float eps, int dtype, void* stream) {
  SANA_REQUIRE(q && k && v && log_decay && state && out, "sana_la_decay: null pointer");
  SANA_REQUIRE(B > 0 && B <= 65535 && N > 0 && N < ((int64_t)1 << 30), "sana_la_decay: B must be in [1, 65535], N in [1, 2^30)");
  int rc = ld_check("sana_la_decay", ldq, ldk, ldv, ldo, H, Hk, D, dtype, q, k, v, out, relu, eps);
  if (rc) return rc;
  SANA_REQUIRE(aligned16(state) && aligned16(prior) && aligned16(workspace), "sana_la_decay: alignment");
  SANA_REQUIRE(prior != state, "sana_la_decay: prior and state must be different buffers");
  SANA_REQUIRE(workspace || workspace_bytes == 0, "sana_la_decay: null workspace");
  LdArgs a = {q, k, v, ldq, ldk, ldv, log_decay, prior, lengths, static_cast<float*>(workspace), state, out, ldo, (int)N, (int)H,
              (int)(H / Hk), 0, 0, 0, scale, eps, relu ? 1 : 0, eps >= 0.f ? 1 : 0, 0};
  LD_DISPATCH(D, return (launch_decay<HD>(a, B, dtype, workspace_bytes, static_cast<cudaStream_t>(stream))));
  return SANA_ERR_INVALID;
}

extern "C" int sana_la_decay_step(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, const float* log_decay,
                                  float* state, int64_t pool, const int32_t* slots, void* out, int64_t ldo, int64_t B, int64_t H,
                                  int64_t Hk, int64_t D, float scale, int relu, float eps, int dtype, void* stream) {
  SANA_REQUIRE(q && k && v && log_decay && state && out, "sana_la_decay_step: null pointer");
  SANA_REQUIRE(B > 0 && B <= 65535, "sana_la_decay_step: B must be in [1, 65535]");
  SANA_REQUIRE(pool > 0 && pool < ((int64_t)1 << 31) && (slots || pool >= B), "sana_la_decay_step: the state holds too few sequences");
  int rc = ld_check("sana_la_decay_step", ldq, ldk, ldv, ldo, H, Hk, D, dtype, q, k, v, out, relu, eps);
  if (rc) return rc;
  SANA_REQUIRE(aligned16(state), "sana_la_decay_step: alignment");
  LdStepArgs a = {q, k, v, ldq, ldk, ldv, log_decay, state, slots, out, ldo, (int)H, (int)(H / Hk), (int)pool, scale, eps,
                  relu ? 1 : 0, eps >= 0.f ? 1 : 0};
  LD_DISPATCH(D, return (launch_decay_step<HD>(a, B, dtype, static_cast<cudaStream_t>(stream))));
  return SANA_ERR_INVALID;
}
