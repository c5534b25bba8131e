// What the kernels of ktb200_latent_attn share: the plan that latent_plan_kernel makes of the call's portions, and small helpers.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include "common.cuh"
#include "umma.cuh"

namespace ktb {

constexpr int kLatent = 512, kLatentRot = 64, kLatentRow = kLatent + kLatentRot, kLatentTile = 128;      // rows of a sequence begin at multiples of kLatentTile
// the plan, ints: the rows of all sequences, the heads of a pass, query tiles, whether a row holds what is not finite; from kPlanSeqs on the first row of each portion and one more, then its keys (0: none, or not there), then the
// tiles (int4, 16-byte aligned: first token, tokens, position of the first, portion)
constexpr int kPlanRows = 0, kPlanHeads = 1, kPlanTiles = 2, kPlanBad = 3, kPlanSeqs = 4, kPlanTokens = 256;      // kPlanTokens: of a query tile
__host__ __device__ inline long plan_tiles_at(int n_seqs) { return ((long)kPlanSeqs + 2 * n_seqs + 1 + 3) / 4 * 4; }

__device__ __forceinline__ uint32_t latent_pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float latent_exp2(float x) {      // one instruction; 2^-inf = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace ktb
