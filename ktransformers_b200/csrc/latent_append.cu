// The append to the paged latent cache (ktb200_latent_append): rotation of all heads' rotated query columns and of the key's, the norm of the latent, the row of the token's page.
//     (a, b) -> gain (a cos x - b sin x, b cos x + a sin x), x = position * frequency;  c / sqrt(mean c^2 + eps) * weight;  one rounding each
// Angles are fp64 up to their remainder of whole turns (in 32 bits a position of 100,000 loses 2^-8 of a radian), everything else fp32.
// Bound by instructions (2000 tokens of 128 heads: 10.6 M of warps, 165 for 32 runs of 8 columns, issue slots 67 % busy; 12 portions of 16 heads: 25.3 M, 72 %) and, for its bytes, by the rotated query
// columns (16 KB a token each way with 128 heads of 64: 2000 tokens 16.0 us, 4.4 TB/s); a decode step by the chain launch, position, angle, store (3.6 us).
// Split: the first CTAs take a latent row a warp; the others some heads of a token, or all heads of up to eight, four runs of 8 columns a thread (a load and a store of 16 bytes each), which are
// loaded ahead of the angles.  (A token a CTA, its loads behind the angles and layouts chosen at run time: 2000 tokens 21 us, 12 portions of 16 heads 75, now 34.)
#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>

#include "common.cuh"

namespace ktb {

constexpr int kLaThreads = 128, kLaLatents = kLaThreads / 32, kLaMaxPairs = 128, kLaAhead = 4, kLaTokens = 8;      // items that a thread has on their way; tokens of a CTA at most

struct LatentAppend {
    ktb200_latent_append_params p;
    int n_tokens, latent_ctas, slices, per, toks;      // CTAs of latent rows; CTAs a token's heads are cut into, the heads of one, the tokens of one
};

// whether token t is in one of the portions that are there, as one is not that reaches past the call's tokens (called by a whole warp)
__device__ __forceinline__ bool latent_in_portion(const ktb200_latent_append_params& p, int n_tokens, int t) {
    bool in = false;
    for (int s = threadIdx.x & 31; s < p.n_seqs; s += 32) {
        const int first = p.seqs[s], count = p.seqs[p.seqs_stride + s];
        in |= first >= 0 && t >= first && t - first < count && count <= n_tokens - first;
    }
    return __any_sync(0xffffffffu, in);
}
__device__ __forceinline__ float2 latent_turn(const ktb200_latent_append_params& p, int t, int i) {
    constexpr double kTurns = 0.15915494309189533577;      // 1 / (2 pi)
    const double x = (double)(p.angle_pos ? p.angle_pos[t] : p.pos[t]) * p.inv_freq[i] * kTurns;
    float s, c;
    sincospif((float)(2.0 * (x - rint(x))), &s, &c);
    return make_float2(c * p.rot_gain, s * p.rot_gain);
}
__device__ __forceinline__ float latent_value(const __nv_bfloat16* x, int i) { return __bfloat162float(x[i]); }
// One head's (or the key's) rotated part, in items: VEC: 8 columns, rot_dims a multiple of 8, 16-byte aligned; otherwise one pair or one column that is not turned
template <bool VEC> __device__ __forceinline__ int latent_items(const ktb200_latent_append_params& p) { return VEC ? p.rot_dim / 8 : p.rot_dims / 2 + p.rot_dim - p.rot_dims; }
// LAYOUT 0: columns 2 i and 2 i + 1 turn in place; 1: they come out at i and i + rot_dims / 2; 2: i and i + rot_dims / 2 turn in place
template <int LAYOUT> __device__ __forceinline__ uint4 latent_load(const __nv_bfloat16* src, int item, int half) {
    if (LAYOUT < 2 || 4 * item >= half) return *reinterpret_cast<const uint4*>(src + 8 * item);
    const uint2 a = *reinterpret_cast<const uint2*>(src + 4 * item), b = *reinterpret_cast<const uint2*>(src + half + 4 * item);
    return make_uint4(a.x, a.y, b.x, b.y);
}
template <int LAYOUT> __device__ __forceinline__ void latent_rotate(const float2* cs, uint4 u, __nv_bfloat16* dst, int item, int half) {      // cs: the token's cosines and sines
    if (4 * item >= half) { *reinterpret_cast<uint4*>(dst + 8 * item) = u; return; }
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    float x[4], y[4];
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
        const float4 t = *reinterpret_cast<const float4*>(cs + 4 * item + k);      // of two pairs
#pragma unroll
        for (int e = 0; e < 2; e++) {
            // halves: words 0, 1 hold the first of the pairs, 2, 3 the second; else a word holds a pair
            const uint32_t f = LAYOUT == 2 ? w[k >> 1] : w[k + e], g = LAYOUT == 2 ? w[2 + (k >> 1)] : f;
            const float a = __uint_as_float(LAYOUT == 2 && e ? f & 0xffff0000u : f << 16), b = __uint_as_float(LAYOUT == 2 && !e ? g << 16 : g & 0xffff0000u), c = e ? t.z : t.x, d = e ? t.w : t.y;
            x[k + e] = a * c - b * d;
            y[k + e] = b * c + a * d;
        }
    }
    auto pack = [](float lo, float hi) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    };
    if (LAYOUT > 0) {
        *reinterpret_cast<uint2*>(dst + 4 * item) = make_uint2(pack(x[0], x[1]), pack(x[2], x[3]));
        *reinterpret_cast<uint2*>(dst + half + 4 * item) = make_uint2(pack(y[0], y[1]), pack(y[2], y[3]));
    } else {
        *reinterpret_cast<uint4*>(dst + 8 * item) = make_uint4(pack(x[0], y[0]), pack(x[1], y[1]), pack(x[2], y[2]), pack(x[3], y[3]));
    }
}
__device__ __forceinline__ void latent_rotate_one(const ktb200_latent_append_params& p, const float2* cs, const __nv_bfloat16* src, __nv_bfloat16* dst, int item) {      // not VEC
    const int half = p.rot_dims / 2;
    if (item >= half) { dst[half + item] = src[half + item]; return; }
    const int i0 = p.rot_layout ? item : 2 * item, i1 = p.rot_layout ? item + half : 2 * item + 1;
    const int o0 = p.rot_layout || p.rot_split ? item : i0, o1 = p.rot_layout || p.rot_split ? item + half : i1;
    const float a = latent_value(src, i0), b = latent_value(src, i1);
    const float2 t = cs[item];
    dst[o0] = __float2bfloat16_rn(a * t.x - b * t.y);
    dst[o1] = __float2bfloat16_rn(b * t.x + a * t.y);
}

// VEC: rows, heads and turned columns in whole 16 bytes.  ITEMS: of a head, where they are known (0: not)
template <bool VEC, int ITEMS, int LAYOUT> __global__ void __launch_bounds__(kLaThreads) latent_append_kernel(const LatentAppend a) {
    const ktb200_latent_append_params& p = a.p;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, width = p.kv_rank + p.rot_dim, half = p.rot_dims / 2, items = ITEMS ? ITEMS : latent_items<VEC>(p);
    __shared__ __align__(16) float2 cs[kLaTokens][kLaMaxPairs];
    __shared__ int there[kLaTokens];
    griddep_launch_dependents();
    griddep_wait();
    if ((int)blockIdx.x < a.latent_ctas) {      // ---------------------------------------------- a warp: one token's latent and key part
        const int t = blockIdx.x * kLaLatents + warp;
        if (t >= a.n_tokens) return;
        const __nv_bfloat16* row = (const __nv_bfloat16*)p.kva + (long)t * p.kva_stride;
        const __nv_bfloat16* weight = (const __nv_bfloat16*)p.norm_weight;
        const int pieces = p.kv_rank / 8;
        uint4 held[2];      // the first 512 columns, on their way while the token's page is looked up
        if (VEC)
#pragma unroll
            for (int i = 0; i < 2; i++) held[i] = lane + 32 * i < pieces ? reinterpret_cast<const uint4*>(row)[lane + 32 * i] : make_uint4(0, 0, 0, 0);
        const int pos = p.pos[t], slot = p.slot[t];
        for (int i = lane; i < half; i += 32) cs[warp][i] = latent_turn(p, t, i);
        const int column = pos / p.page_size;      // (a position behind the last column has no row: nothing to write to)
        if (!latent_in_portion(p, a.n_tokens, t) || pos < 0 || column >= p.max_pages || (unsigned)slot >= (unsigned)p.n_slots) return;
        const int page = p.page_table[(long)slot * p.max_pages + column];
        if ((unsigned)page >= (unsigned)p.n_pages) return;
        __nv_bfloat16* dst = (__nv_bfloat16*)p.cache + ((long)page * p.page_size + pos % p.page_size) * width;
        float sum = 0.f;
        auto squares = [&](uint4 u) {
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float x = __uint_as_float(w[k] << 16), y = __uint_as_float(w[k] & 0xffff0000u);
                sum = fmaf(x, x, fmaf(y, y, sum));
            }
        };
        if (VEC) {
            squares(held[0]);
            squares(held[1]);
            for (int i = lane + 64; i < pieces; i += 32) squares(reinterpret_cast<const uint4*>(row)[i]);
        } else {
            for (int i = lane; i < p.kv_rank; i += 32) sum = fmaf(latent_value(row, i), latent_value(row, i), sum);
        }
        const float inv = 1.0f / sqrtf(warp_sum(sum) / (float)p.kv_rank + p.eps);
        __syncwarp();
        auto normed = [&](int i, uint4 u) {
            const uint4 g = reinterpret_cast<const uint4*>(weight)[i];
            const uint32_t w[4] = {u.x, u.y, u.z, u.w}, f[4] = {g.x, g.y, g.z, g.w};
            uint32_t o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(w[k] << 16) * inv * __uint_as_float(f[k] << 16),
                                                               __uint_as_float(w[k] & 0xffff0000u) * inv * __uint_as_float(f[k] & 0xffff0000u));
                o[k] = *reinterpret_cast<const uint32_t*>(&v);
            }
            reinterpret_cast<uint4*>(dst)[i] = make_uint4(o[0], o[1], o[2], o[3]);
        };
        if (VEC) {
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (lane + 32 * i < pieces) normed(lane + 32 * i, held[i]);
            for (int i = lane + 64; i < pieces; i += 32) normed(i, reinterpret_cast<const uint4*>(row)[i]);
            for (int i = lane; i < items; i += 32) latent_rotate<LAYOUT>(cs[warp], latent_load<LAYOUT>(row + p.kv_rank, i, half), dst + p.kv_rank, i, half);
        } else {
            for (int i = lane; i < p.kv_rank; i += 32) dst[i] = __float2bfloat16_rn(latent_value(row, i) * inv * latent_value(weight, i));
            for (int i = lane; i < items; i += 32) latent_rotate_one(p, cs[warp], row + p.kv_rank, dst + p.kv_rank, i);
        }
        return;
    }
    // ------------------------------------------------------------------------------------------ a CTA: some of the heads of one to eight tokens
    const int b = blockIdx.x - a.latent_ctas, t0 = b / a.slices * a.toks, h0 = (b % a.slices) * a.per, heads = min(a.per, p.heads - h0), toks = min(a.toks, a.n_tokens - t0), hw = p.nope_dim + p.rot_dim;
    const int n = toks * heads * items;
    const __nv_bfloat16* q = (const __nv_bfloat16*)p.q + (long)t0 * p.q_stride + (long)h0 * hw + p.nope_dim;
    __nv_bfloat16* out = (__nv_bfloat16*)p.q_rot + ((long)t0 * p.heads + h0) * p.rot_dim;
    // the thread's items: item x % items of head x / items % heads of token x / items / heads, x = thread, thread + threads, ..  (ITEMS divides the threads: its item stays the same)
    struct Place { int token, head, item; };
    auto first = [&](int x) { const int h = x / items; return Place{h / heads, h % heads, x - h * items}; };
    auto next = [&](Place& at, int x) {
        if (!ITEMS) { at = first(x); return; }
        for (at.head += kLaThreads / (ITEMS ? ITEMS : 1); at.head >= heads; at.head -= heads) at.token++;
    };
    uint4 held[kLaAhead];
    Place in = first(threadIdx.x), at = in;
    auto load = [&](int u0) {
#pragma unroll
        for (int i = 0; i < kLaAhead; i++) {
            const int u = u0 + i * kLaThreads + threadIdx.x;
            if (u < n) held[i] = latent_load<LAYOUT>(q + (long)in.token * p.q_stride + in.head * hw, in.item, half);
            next(in, u + kLaThreads);
        }
    };
    if (VEC) load(0);      // (on their way while the angles are made)
    for (int i = threadIdx.x; i < toks * half; i += kLaThreads) cs[i / half][i % half] = latent_turn(p, t0 + i / half, i % half);
    for (int k = warp; k < toks; k += kLaThreads / 32) {
        const bool mine = latent_in_portion(p, a.n_tokens, t0 + k);
        if (lane == 0) there[k] = mine;
    }
    __syncthreads();
    if (VEC) {
        for (int u0 = 0; u0 < n; u0 += kLaAhead * kLaThreads) {
            if (u0 > 0) load(u0);
#pragma unroll
            for (int i = 0; i < kLaAhead; i++) {
                const int u = u0 + i * kLaThreads + threadIdx.x;
                if (u < n && there[at.token]) latent_rotate<LAYOUT>(cs[at.token], held[i], out + ((long)at.token * p.heads + at.head) * p.rot_dim, at.item, half);
                next(at, u + kLaThreads);
            }
        }
    } else {
        for (int u = threadIdx.x; u < n; u += kLaThreads) {
            at = first(u);
            if (there[at.token]) latent_rotate_one(p, cs[at.token], q + (long)at.token * p.q_stride + at.head * hw, out + ((long)at.token * p.heads + at.head) * p.rot_dim, at.item);
        }
    }
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
    // a CTA takes what its threads have on their way at once (kLaAhead items each): some of a token's heads, or the heads of up to eight tokens.  A step of few tokens is cut further, down to one
    // round of threads, until it fills the SMs
    const long items = (long)p->heads * std::max(p->rot_dim / 8, 1), most = kLaThreads * kLaAhead, sms = num_sms(device);
    a.slices = (int)std::max((items + most - 1) / most, std::min((items + kLaThreads - 1) / kLaThreads, sms * 4 / n_tokens));
    a.per = (p->heads + a.slices - 1) / a.slices;
    a.slices = (p->heads + a.per - 1) / a.per;
    a.toks = a.slices > 1 ? 1 : (int)std::max(1L, std::min({most / items, (long)kLaTokens, n_tokens / (sms * 2)}));
    const long grid = a.latent_ctas + (n_tokens + a.toks - 1) / a.toks * (long)a.slices;
    if (grid > 0x7fffffffL) { set_error("latent_append: too many tokens"); return KTB200_EINVAL; }
    auto pick = [&](auto items) {
        constexpr int I = decltype(items)::value;
        return p->rot_layout ? latent_append_kernel<true, I, 2> : p->rot_split ? latent_append_kernel<true, I, 1> : latent_append_kernel<true, I, 0>;
    };
    const auto kernel = !vec ? latent_append_kernel<false, 0, 0> : p->rot_dim == 64 ? pick(std::integral_constant<int, 8>()) : pick(std::integral_constant<int, 0>());
    KTB_CUDA_CHECK(launch_pdl(kernel, dim3((unsigned)grid), dim3(kLaThreads), (size_t)0, (cudaStream_t)stream, a));
    count_launch();
    return KTB200_OK;
}
