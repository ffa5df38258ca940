// Arguments and small helpers shared by the kernels of the decaying linear attention (la_decay.cu, la_decay_tc.cu).
#pragma once
#include "la_plan.cuh"
#include "tc_common.cuh"

namespace sana {

struct LdArgs {
  const void *q, *k, *v;
  int64_t ldq, ldk, ldv;
  const float* log_decay;    // [H]
  const float* prior;        // [B, H, D+1, D] or null
  const int* lengths;        // [B] or null
  float* partial;            // [B, npart, H, D+1, D]: what each token segment adds to the state
  float* state;              // [B, H, D+1, D]
  void* out;
  int64_t ldo;
  int N, H, group;           // group = query heads per key/value head
  int seg_len, nseg, npart;
  float scale, eps;
  int relu, normalise;
  int wide_rows;             // output rows are 32-byte aligned
};

__device__ __forceinline__ float ld_power(float g, int n) { return n == 0 ? 1.f : expf(g * (float)n); }

__device__ __forceinline__ uint32_t ld_relu2(uint32_t r) {  // a NaN stays one
  const __nv_bfloat162 x = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&r), __floats2bfloat162_rn(0.f, 0.f));
  return *reinterpret_cast<const uint32_t*>(&x);
}
// the bf16 pair nearest (a, b), and what it leaves of them
__device__ __forceinline__ uint32_t ld_split(float& a, float& b) {
  const uint32_t p = pack_bf16(a, b);
  a -= bf16_lo(p);
  b -= bf16_hi(p);
  return p;
}

// Split of a sequence into nseg token segments of seg_len tokens (whole chunks; the last may be shorter).  The rules that
// choose it: ld_tc_plan, and ld_plan for fp32.
struct LdPlan {
  int seg_len, nseg;
};

// tcgen05 kernels (la_decay_tc.cu); D a multiple of 16 in [16, 128]
LdPlan ld_tc_plan(int64_t B, int64_t N, int64_t H, int64_t D, bool ragged, int* npart);  // ragged: lengths are given
int launch_decay_tc(LdArgs& a, int64_t B, int64_t D, cudaStream_t st);

}  // namespace sana
