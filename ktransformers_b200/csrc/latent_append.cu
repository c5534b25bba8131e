// The append to the paged latent cache (ktb200_latent_append): rotation of all heads' rotated query columns and of the key's, the norm of the latent, the row of the token's page.
//     (a, b) -> gain (a cos x - b sin x, b cos x + a sin x), x = position * frequency;  c / sqrt(mean c^2 + eps) * weight;  one rounding each
// Angles are fp64 up to their remainder of whole turns (in 32 bits a position of 100,000 loses 2^-8 of a radian), everything else fp32.
// Bound by the bytes of the rotated query columns (16 KB a token each way with 128 heads of 64); a decode step by the chain launch, position, angle, store.
// Split: the first CTAs take a latent row a warp, the others a token's heads, 8 columns a thread (a load and a store of 16 bytes).
#include <algorithm>

#include <cuda_bf16.h>

#include "common.cuh"

namespace ktb {

constexpr int kLaThreads = 256, kLaLatents = kLaThreads / 32, kLaMaxPairs = 128;

struct LatentAppend {
    ktb200_latent_append_params p;
    int n_tokens, latent_ctas, slices, per;      // CTAs of latent rows; CTAs a token's heads are cut into, and the heads of one
};

// whether token t is in one of the portions (called by a whole warp)
__device__ __forceinline__ bool latent_in_portion(const int* seqs, int stride, int n_seqs, int t) {
    bool in = false;
    for (int s = threadIdx.x & 31; s < n_seqs; s += 32) {
        const int first = seqs[s];
        in |= t >= first && t - first < seqs[stride + s];
    }
    return __any_sync(0xffffffffu, in);
}
__device__ __forceinline__ float2 latent_turn(const ktb200_latent_append_params& p, int t, int i) {
    constexpr double kTurn = 6.283185307179586477;
    const double x = (double)(p.angle_pos ? p.angle_pos[t] : p.pos[t]) * p.inv_freq[i];
    float s, c;
    sincosf((float)(x - rint(x / kTurn) * kTurn), &s, &c);
    return make_float2(c * p.rot_gain, s * p.rot_gain);
}
__device__ __forceinline__ float latent_value(const __nv_bfloat16* x, int i) { return __bfloat162float(x[i]); }
// columns `c` .. of one head's (or the key's) rotated part, from src to dst; cs: the token's cosines and sines.  VEC: 8 columns, rot_dims a multiple of 8, 16-byte aligned;
// otherwise one pair or one column that is not turned
template <bool VEC> __device__ __forceinline__ int latent_items(const ktb200_latent_append_params& p) { return VEC ? p.rot_dim / 8 : p.rot_dims / 2 + p.rot_dim - p.rot_dims; }
template <bool VEC> __device__ __forceinline__ void latent_rotate(const ktb200_latent_append_params& p, const float2* cs, const __nv_bfloat16* src, __nv_bfloat16* dst, int item) {
    const int half = p.rot_dims / 2, turned = VEC ? p.rot_dims / 8 : half;
    if (item >= turned) {
        if (VEC) *reinterpret_cast<uint4*>(dst + 8 * item) = *reinterpret_cast<const uint4*>(src + 8 * item);
        else dst[p.rot_dims + item - turned] = src[p.rot_dims + item - turned];
        return;
    }
    if (!VEC) {
        const int i0 = p.rot_layout ? item : 2 * item, i1 = p.rot_layout ? item + half : 2 * item + 1;
        const int o0 = p.rot_layout || p.rot_split ? item : i0, o1 = p.rot_layout || p.rot_split ? item + half : i1;
        const float a = latent_value(src, i0), b = latent_value(src, i1);
        const float2 t = cs[item];
        dst[o0] = __float2bfloat16_rn(a * t.x - b * t.y);
        dst[o1] = __float2bfloat16_rn(b * t.x + a * t.y);
        return;
    }
    float a[4], b[4];
    if (p.rot_layout) {
        const uint2 u = *reinterpret_cast<const uint2*>(src + 4 * item), v = *reinterpret_cast<const uint2*>(src + half + 4 * item);
        const uint32_t w[4] = {u.x, u.y, v.x, v.y};
#pragma unroll
        for (int k = 0; k < 4; k++) (k < 2 ? a[2 * k] : b[2 * k - 4]) = __uint_as_float(w[k] << 16), (k < 2 ? a[2 * k + 1] : b[2 * k - 3]) = __uint_as_float(w[k] & 0xffff0000u);
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(src + 8 * item);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; k++) a[k] = __uint_as_float(w[k] << 16), b[k] = __uint_as_float(w[k] & 0xffff0000u);
    }
    float x[4], y[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float2 t = cs[4 * item + k];
        x[k] = a[k] * t.x - b[k] * t.y;
        y[k] = b[k] * t.x + a[k] * t.y;
    }
    auto pack = [](float lo, float hi) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    };
    if (p.rot_layout || p.rot_split) {
        *reinterpret_cast<uint2*>(dst + 4 * item) = make_uint2(pack(x[0], x[1]), pack(x[2], x[3]));
        *reinterpret_cast<uint2*>(dst + half + 4 * item) = make_uint2(pack(y[0], y[1]), pack(y[2], y[3]));
    } else {
        *reinterpret_cast<uint4*>(dst + 8 * item) = make_uint4(pack(x[0], y[0]), pack(x[1], y[1]), pack(x[2], y[2]), pack(x[3], y[3]));
    }
}

// VEC: rows, heads and turned columns in whole 16 bytes
template <bool VEC> __global__ void __launch_bounds__(kLaThreads) latent_append_kernel(const LatentAppend a) {
    const ktb200_latent_append_params& p = a.p;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, width = p.kv_rank + p.rot_dim, half = p.rot_dims / 2;
    __shared__ float2 cs[kLaLatents][kLaMaxPairs];
    griddep_launch_dependents();
    griddep_wait();
    if ((int)blockIdx.x < a.latent_ctas) {      // ---------------------------------------------- a warp: one token's latent and key part
        const int t = blockIdx.x * kLaLatents + warp;
        if (t >= a.n_tokens || !latent_in_portion(p.seqs, p.seqs_stride, p.n_seqs, t)) return;
        const int pos = p.pos[t], slot = p.slot[t];
        if (pos < 0 || (unsigned)slot >= (unsigned)p.n_slots) return;
        const int page = p.page_table[(long)slot * p.max_pages + (pos / p.page_size) % p.max_pages];
        if ((unsigned)page >= (unsigned)p.n_pages) return;
        const __nv_bfloat16* row = (const __nv_bfloat16*)p.kva + (long)t * p.kva_stride;
        const __nv_bfloat16* weight = (const __nv_bfloat16*)p.norm_weight;
        __nv_bfloat16* dst = (__nv_bfloat16*)p.cache + ((long)page * p.page_size + pos % p.page_size) * width;
        for (int i = lane; i < half; i += 32) cs[warp][i] = latent_turn(p, t, i);
        float sum = 0.f;
        if (VEC) {
            for (int i = lane; i < p.kv_rank / 8; i += 32) {
                const uint4 u = reinterpret_cast<const uint4*>(row)[i];
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float x = __uint_as_float(w[k] << 16), y = __uint_as_float(w[k] & 0xffff0000u);
                    sum = fmaf(x, x, fmaf(y, y, sum));
                }
            }
        } else {
            for (int i = lane; i < p.kv_rank; i += 32) sum = fmaf(latent_value(row, i), latent_value(row, i), sum);
        }
        const float inv = 1.0f / sqrtf(warp_sum(sum) / (float)p.kv_rank + p.eps);
        __syncwarp();
        if (VEC) {
            for (int i = lane; i < p.kv_rank / 8; i += 32) {      // (in L1 by now)
                const uint4 u = reinterpret_cast<const uint4*>(row)[i], g = reinterpret_cast<const uint4*>(weight)[i];
                const uint32_t w[4] = {u.x, u.y, u.z, u.w}, f[4] = {g.x, g.y, g.z, g.w};
                uint32_t o[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(w[k] << 16) * inv * __uint_as_float(f[k] << 16),
                                                                   __uint_as_float(w[k] & 0xffff0000u) * inv * __uint_as_float(f[k] & 0xffff0000u));
                    o[k] = *reinterpret_cast<const uint32_t*>(&v);
                }
                reinterpret_cast<uint4*>(dst)[i] = make_uint4(o[0], o[1], o[2], o[3]);
            }
        } else {
            for (int i = lane; i < p.kv_rank; i += 32) dst[i] = __float2bfloat16_rn(latent_value(row, i) * inv * latent_value(weight, i));
        }
        for (int i = lane; i < latent_items<VEC>(p); i += 32) latent_rotate<VEC>(p, cs[warp], row + p.kv_rank, dst + p.kv_rank, i);
        return;
    }
    // ------------------------------------------------------------------------------------------ a CTA: some of one token's heads
    const int b = blockIdx.x - a.latent_ctas, t = b / a.slices, h0 = (b % a.slices) * a.per, heads = min(a.per, p.heads - h0);
    const bool in = latent_in_portion(p.seqs, p.seqs_stride, p.n_seqs, t);      // (every warp for itself)
    if (!in) return;
    for (int i = threadIdx.x; i < half; i += kLaThreads) cs[0][i] = latent_turn(p, t, i);
    __syncthreads();
    const int items = latent_items<VEC>(p), hw = p.nope_dim + p.rot_dim;
    const __nv_bfloat16* src = (const __nv_bfloat16*)p.q + (long)t * p.q_stride + (long)h0 * hw + p.nope_dim;
    __nv_bfloat16* dst = (__nv_bfloat16*)p.q_rot + ((long)t * p.heads + h0) * p.rot_dim;
#pragma unroll 4
    for (int u = threadIdx.x; u < heads * items; u += kLaThreads) latent_rotate<VEC>(p, cs[0], src + (long)(u / items) * hw, dst + (long)(u / items) * p.rot_dim, u % items);
}

}  // namespace ktb

using namespace ktb;

extern "C" int ktb200_latent_append(const ktb200_latent_append_params* p, int n_tokens, void* stream) {
    if (!p || p->heads <= 0 || p->nope_dim < 0 || p->kv_rank <= 0 || p->rot_dim < 0 || p->page_size <= 0 || p->max_pages <= 0 || p->n_slots <= 0 || p->n_pages <= 0 || p->n_seqs < 0) {
        set_error("latent_append: bad sizes");
        return KTB200_EINVAL;
    }
    if (p->rot_dims < 0 || p->rot_dims > p->rot_dim || p->rot_dims % 2 || p->rot_dims > 2 * kLaMaxPairs || p->rot_layout < 0 || p->rot_layout > 1 || (p->rot_dims > 0 && !p->inv_freq)) {
        set_error("latent_append: rot_dims %d of %d columns: an even number up to %d, with inv_freq, in layout 0 or 1", p->rot_dims, p->rot_dim, 2 * kLaMaxPairs);
        return KTB200_EINVAL;
    }
    if (p->q_stride < (long)p->heads * (p->nope_dim + p->rot_dim) || p->kva_stride < p->kv_rank + p->rot_dim) { set_error("latent_append: rows overlap"); return KTB200_EINVAL; }
    if (n_tokens <= 0 || p->n_seqs == 0) return KTB200_OK;
    if (!p->q || !p->kva || !p->norm_weight || !p->pos || !p->slot || !p->seqs || !p->page_table || !p->cache || (!p->q_rot && p->rot_dim > 0)) { set_error("latent_append: null pointer"); return KTB200_EINVAL; }
    int device = 0;
    KTB_CUDA_CHECK(cudaGetDevice(&device));
    LatentAppend a;
    a.p = *p;
    a.n_tokens = n_tokens;
    a.latent_ctas = (n_tokens + kLaLatents - 1) / kLaLatents;
    const int hw = p->nope_dim + p->rot_dim;
    const bool vec = p->rot_dims % 8 == 0 && p->rot_dim % 8 == 0 && p->nope_dim % 8 == 0 && p->kv_rank % 8 == 0 && p->q_stride % 8 == 0 && p->kva_stride % 8 == 0 && hw % 8 == 0 &&
                     (((uintptr_t)p->q | (uintptr_t)p->kva | (uintptr_t)p->norm_weight | (uintptr_t)p->cache | (uintptr_t)p->q_rot) & 15) == 0;
    // a token's heads are cut so far that a step of few tokens fills the SMs; in parts of at least one round of the CTA's threads
    const long rounds = ((long)p->heads * std::max(p->rot_dim / 8, 1) + kLaThreads - 1) / kLaThreads;
    a.slices = (int)std::max(1L, std::min(rounds, (long)num_sms(device) * 4 / n_tokens));
    a.per = (p->heads + a.slices - 1) / a.slices;
    a.slices = (p->heads + a.per - 1) / a.per;
    const long grid = a.latent_ctas + (long)n_tokens * a.slices;
    if (grid > 0x7fffffffL) { set_error("latent_append: too many tokens"); return KTB200_EINVAL; }
    KTB_CUDA_CHECK(launch_pdl(vec ? latent_append_kernel<true> : latent_append_kernel<false>, dim3((unsigned)grid), dim3(kLaThreads), (size_t)0, (cudaStream_t)stream, a));
    count_launch();
    return KTB200_OK;
}
