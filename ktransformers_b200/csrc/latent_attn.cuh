// What the kernels of ktb200_latent_attn share: the plan that latent_plan_kernel makes of the call's portions, and small helpers.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include "common.cuh"
#include "umma.cuh"

namespace ktb {

constexpr int kLatent = 512, kLatentRot = 64, kLatentRow = kLatent + kLatentRot, kLatentTile = 128;      // rows of a sequence begin at multiples of kLatentTile
// the plan, ints: the rows of all sequences, the heads of a pass, query tiles, what rows are odd (kOddBad: one holds what is not finite, kOddGone: the page of a key is not
// there); from kPlanSeqs on the first row of each portion and one more, then its keys (0: none, or not there), then the
// tiles (int4, 16-byte aligned: first token, tokens, position of the first, portion)
constexpr int kPlanRows = 0, kPlanHeads = 1, kPlanTiles = 2, kPlanOdd = 3, kPlanSeqs = 4, kPlanTokens = 256;      // kPlanTokens: of a query tile
constexpr int kOddBad = 1, kOddGone = 2;
__host__ __device__ inline long plan_tiles_at(int n_seqs) { return ((long)kPlanSeqs + 2 * n_seqs + 1 + 3) / 4 * 4; }

// positions that have a column of the page table: keys from there on are not there, and tokens at such positions see those that are
__host__ __device__ inline int latent_room(const ktb200_latent_attn_params& p) {
    const long n = (long)p.max_pages * p.page_size;
    return n < 0x7fffff00L ? (int)n : 0x7fffff00;
}
// A portion as all kernels of both forms see it; count 0: not there, as one is that reaches past the call's tokens or whose first token's position or slot is not there
struct LatentPortion { int first, count, pos, slot, end; };      // end: keys that its last token sees
__device__ __forceinline__ LatentPortion latent_portion(const ktb200_latent_attn_params& p, int n_tokens, int s) {
    LatentPortion q{p.seqs[s], p.seqs[p.seqs_stride + s], 0, 0, 0};
    if (q.count <= 0 || q.first < 0 || q.first > n_tokens - q.count) { q.count = 0; return q; }
    q.pos = p.pos[q.first];
    q.slot = p.slot[q.first];
    if (q.pos < 0 || q.pos > 0x7fffff00 - q.count || (unsigned)q.slot >= (unsigned)p.n_slots) { q.count = 0; return q; }
    q.end = min(q.pos + q.count, latent_room(p));
    return q;
}
__device__ __forceinline__ uint32_t latent_pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// A warp copies one cache row, or zeros where it is not there.  With `clean` a latent that holds a number that is not finite becomes zeros, and the answer is true: whoever sees the row is to be
// NaN, and whoever does not must not meet it (0 x NaN).  The rotated part stays: what it holds reaches the scores alone
__device__ __forceinline__ bool latent_copy_row(const __nv_bfloat16* src, bool there, __nv_bfloat16* dst, bool clean) {
    const int lane = threadIdx.x & 31;
    uint4 v[3];
    bool finite = true;
#pragma unroll
    for (int c = 0; c < 3; c++) {
        v[c] = there && lane + 32 * c < kLatentRow / 8 ? reinterpret_cast<const uint4*>(src)[lane + 32 * c] : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
        for (int k = 0; k < 4; k++) finite &= c == 2 || ((w[k] & 0x7f800000u) != 0x7f800000u && (w[k] & 0x7f80u) != 0x7f80u);
    }
    const bool whole = __all_sync(0xffffffffu, finite) || !clean;
#pragma unroll
    for (int c = 0; c < 3; c++)
        if (lane + 32 * c < kLatentRow / 8) reinterpret_cast<uint4*>(dst)[lane + 32 * c] = whole || c == 2 ? v[c] : make_uint4(0, 0, 0, 0);
    return !whole;
}
// A sum of weights that is zero where keys are not there: the row sees none and becomes zero.  (Elsewhere all of its scores are -inf, and it is NaN.)  The parts of a row hand it on as -0
constexpr uint32_t kNoKeys = 0x80000000u;
__device__ __forceinline__ float latent_sum(float l, bool gone) { return gone && l == 0.f ? __uint_as_float(kNoKeys) : l; }
__device__ __forceinline__ float latent_inverse(float l) { return __float_as_uint(l) == kNoKeys ? 0.f : 1.f / l; }
// a sector of 32 bytes, from a thread
template <typename T> __device__ __forceinline__ void latent_store32(T* to, const uint32_t* w) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
__device__ __forceinline__ float latent_exp2(float x) {      // one instruction; 2^-inf = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace ktb
