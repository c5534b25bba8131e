// Appending keys and values to the paged e4m3 cache (fp8_cache.cuh), with the norms and the rotation applied on the way (libktb200_seq.so).
//
//   ktb200_fp8_cache_append   proj rows [... q ... k ... v ...]; q and k, head by head: nothing (qk_norm 0), x / sqrt(mean x^2 + eps) (1), the same times one weight per
//                             column (3); then a turn of the first rot_dims columns (pairs of either layout, angle pos * inv_freq[i]).  q to q_out; k and v as
//                             e4m3 codes under one scale per page and head.
//
// The tokens of a portion that fall into one page are appended by one CTA per key/value head, which finds their largest |k| and |v|, makes the block's scales, moves
// the codes of the tokens that the page held before where a scale has grown, and writes the new codes: no other CTA touches the block, so there is nothing to
// order and nothing to add up atomically.  A portion that begins at a page's first token starts its blocks anew (whatever the page held).
// Rotation, norms and scaling are fp32; angles are reduced in fp64.
#include <cuda_bf16.h>

#include <algorithm>

#include "fp8_cache.cuh"

namespace ktb {

constexpr int kAppThreads = 256, kAppWarps = kAppThreads / 32, kAppCols = 8 /* columns of a lane: head sizes up to 256 */, kAppKeep = 96 * 1024;

struct Fp8Append {
    const void* proj;
    long proj_stride;
    int q_off, k_off, v_off, H, G, d, dv, rot_dims, rot_layout;
    const double* inv_freq;
    int qk_norm;
    const void *q_w, *k_w;
    float eps;
    const int *pos, *slot, *seqs;
    int seqs_stride, n_seqs, n_tokens;
    Fp8Pages pages;
    uint8_t *k_codes, *v_codes;
    float* scales;
    void* q_out;
    int kv_ctas, keep, q_tokens, q_heads, q_blocks;
};

// (cos, sin) of pos * freq: the angle and its remainder in 64 bits, sine and cosine of the remainder's fp32 part, corrected by what that left
__device__ __forceinline__ float2 app_turn(int pos, double freq) {
    const double angle = (double)pos * freq, rest = fma(-rint(angle * 0.15915494309189535), 6.283185307179586, angle);
    const float hi = (float)rest, lo = (float)(rest - (double)hi);
    float sn, cs;
    sincosf(hi, &sn, &cs);
    return make_float2(fmaf(-lo, sn, cs), fmaf(lo, cs, sn));
}

// One head's columns of one token, as a warp holds them.  PER > 0: heads of 32 PER columns, a lane's PER of them side by side; PER = 0: any size, columns lane, lane + 32, ..
template <typename T, int PER> struct AppRow {
    static constexpr int N = PER ? PER : kAppCols;
    float x[N];
    __device__ __forceinline__ static int col(int e) { const int lane = threadIdx.x & 31; return PER ? lane * PER + e : lane + 32 * e; }
    __device__ __forceinline__ void load(const T* row, int n) {
        if constexpr (PER == 0) {
#pragma unroll
            for (int e = 0; e < N; e++) x[e] = col(e) < n ? to_f(row[col(e)]) : 0.f;
        } else if constexpr (sizeof(T) == 4) {
            if constexpr (PER == 2) {
                const float2 v = *reinterpret_cast<const float2*>(row + col(0));
                x[0] = v.x; x[1] = v.y;
            } else {
#pragma unroll
                for (int e = 0; e < N; e += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(row + col(e));
                    x[e] = v.x; x[e + 1] = v.y; x[e + 2] = v.z; x[e + 3] = v.w;
                }
            }
        } else {
            uint32_t w[PER / 2];
            if constexpr (PER == 2) w[0] = *reinterpret_cast<const uint32_t*>(row + col(0));
            else if constexpr (PER == 4) { const uint2 v = *reinterpret_cast<const uint2*>(row + col(0)); w[0] = v.x; w[1] = v.y; }
            else { const uint4 v = *reinterpret_cast<const uint4*>(row + col(0)); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
#pragma unroll
            for (int e = 0; e < PER / 2; e++) { x[2 * e] = __uint_as_float(w[e] << 16); x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
        }
    }
    // norm and turn; `turn(i)`: (cos, sin) of pair i
    template <typename Turn> __device__ __forceinline__ void prepare(const T* row, const Fp8Append& a, const T* w, Turn turn) {
        const int lane = threadIdx.x & 31, half = a.rot_dims >> 1;
        float inv = 1.f;
        if (a.qk_norm) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < N; e++) ss = fmaf(x[e], x[e], ss);
            inv = 1.0f / sqrtf(warp_sum(ss) / (float)a.d + a.eps);
#pragma unroll
            for (int e = 0; e < N; e++)
                if (PER || col(e) < a.d) x[e] = a.qk_norm == 3 ? x[e] * inv * to_f(w[col(e)]) : x[e] * inv;
        }
        if (a.rot_dims == 0) return;
        if (a.rot_layout == kRotInterleaved && PER) {
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                const int c = col(e);
                if (c < a.rot_dims) {
                    const float2 t = turn(c >> 1);
                    const float u = x[e], v = x[e + 1];
                    x[e] = u * t.x - v * t.y;
                    x[e + 1] = v * t.x + u * t.y;
                }
            }
        } else if (PER) {      // halves: the partner's lane is half / PER lanes away
            const int step = half / (PER ? PER : 1);
#pragma unroll
            for (int e = 0; e < N; e++) {
                const int c = col(e);
                const bool second = c >= half;
                const float other = __shfl_sync(0xffffffffu, x[e], second ? lane - step : lane + step);
                if (c < a.rot_dims) {
                    const float2 t = turn(second ? c - half : c);
                    x[e] = second ? x[e] * t.x + other * t.y : x[e] * t.x - other * t.y;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < N; e++) {
                const int c = col(e);
                if (c < a.rot_dims) {
                    const int o = rot_partner(c, a.rot_dims, a.rot_layout);
                    const bool second = a.rot_layout == kRotHalves ? c >= half : (c & 1);
                    const float2 t = turn(a.rot_layout == kRotHalves ? (second ? c - half : c) : (c >> 1));
                    float other = to_f(row[o]) * inv;
                    if (a.qk_norm == 3) other *= to_f(w[o]);
                    x[e] = second ? x[e] * t.x + other * t.y : x[e] * t.x - other * t.y;
                }
            }
        }
    }
    __device__ __forceinline__ float top(int n) const {
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < N; e++) m = fmaxf(m, fabsf(x[e]));      // (columns behind a head's last are zero)
        return m;
    }
    __device__ __forceinline__ void store(T* row, int n) const {
        if constexpr (PER == 0) {
#pragma unroll
            for (int e = 0; e < N; e++)
                if (col(e) < n) row[col(e)] = from_f<T>(x[e]);
        } else if constexpr (PER == 2) {
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(row + col(0)) = make_float2(x[0], x[1]);
            else { const __nv_bfloat162 v = __floats2bfloat162_rn(x[0], x[1]); *reinterpret_cast<__nv_bfloat162*>(row + col(0)) = v; }
        } else {
#pragma unroll
            for (int e = 0; e < N; e += 4) store4(row + col(e), make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]));
        }
    }
    __device__ __forceinline__ void store_codes(uint8_t* row, int n, float inv_scale) const {
        if constexpr (PER == 0) {
#pragma unroll
            for (int e = 0; e < N; e++)
                if (col(e) < n) row[col(e)] = (uint8_t)__nv_cvt_float_to_fp8(x[e] * inv_scale, __NV_SATFINITE, __NV_E4M3);
        } else {
            uint32_t w[(PER + 3) / 4] = {};
#pragma unroll
            for (int e = 0; e < N; e += 2)
                w[e / 4] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[e] * inv_scale, x[e + 1] * inv_scale), __NV_SATFINITE, __NV_E4M3) << (8 * (e & 3));
            if constexpr (PER == 2) *reinterpret_cast<uint16_t*>(row + col(0)) = (uint16_t)w[0];
            else if constexpr (PER == 4) *reinterpret_cast<uint32_t*>(row + col(0)) = w[0];
            else *reinterpret_cast<uint2*>(row + col(0)) = make_uint2(w[0], w[1]);
        }
    }
};

// the smallest e with 448 2^e >= top: top = 1.f 2^x, 448 = 1.75 2^8
__device__ __forceinline__ int fp8_exponent(float top) {
    const uint32_t b = __float_as_uint(top);
    const int e = (int)(b >> 23) - 127 - ((b & 0x7fffffu) <= 0x600000u ? 8 : 7);
    return min(kFp8EMax, max(kFp8EMin, e));
}
__device__ __forceinline__ float fp8_power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The codes of `bytes` bytes at p times f (a power of two below one)
__device__ __forceinline__ void fp8_move(uint8_t* p, long bytes, float f) {
    if (((reinterpret_cast<uintptr_t>(p) | bytes) & 3) == 0) {
        for (long i = 4 * (long)threadIdx.x; i < bytes; i += 4 * kAppThreads) {
            uint32_t w = *reinterpret_cast<uint32_t*>(p + i), r = 0;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const __half2_raw v = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * h)), __NV_E4M3);
                const float2 x = __half22float2(__half2(v));
                r |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x.x * f, x.y * f), __NV_SATFINITE, __NV_E4M3) << (16 * h);
            }
            *reinterpret_cast<uint32_t*>(p + i) = r;
        }
    } else {
        for (long i = threadIdx.x; i < bytes; i += kAppThreads) {
            const float x = __half2float(__half(__nv_cvt_fp8_to_halfraw(p[i], __NV_E4M3)));
            p[i] = (uint8_t)__nv_cvt_float_to_fp8(x * f, __NV_SATFINITE, __NV_E4M3);
        }
    }
}

// Blocks [0, kv_ctas): one page's tokens of one portion for one key/value head (the portions' pages in order, heads fastest); the blocks behind them: q_tokens tokens
// times q_heads query heads.
template <typename T, int PER> __global__ void __launch_bounds__(kAppThreads) fp8_append_kernel(const Fp8Append a) {
    using Row = AppRow<T, PER>;
    extern __shared__ __align__(16) float app_smem[];
    __shared__ float tops[2][kAppWarps];
    __shared__ int info[4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ps = a.pages.page_size;
    const T* proj = (const T*)a.proj;
    griddep_launch_dependents();
    griddep_wait();
    if ((int)blockIdx.x >= a.kv_ctas) {
        const int b = blockIdx.x - a.kv_ctas, t0 = (b / a.q_blocks) * a.q_tokens, h0 = (b % a.q_blocks) * a.q_heads, half = a.rot_dims >> 1;
        const int nt = min(a.q_tokens, a.n_tokens - t0), nh = min(a.q_heads, a.H - h0);
        float2* table = reinterpret_cast<float2*>(app_smem);
        for (int i = threadIdx.x; i < nt * half; i += kAppThreads) table[i] = app_turn(a.pos[t0 + i / half], a.inv_freq[i % half]);
        __syncthreads();
        constexpr int U = PER ? 4 : 1;      // units whose loads are in flight together
        for (int u0 = warp * U; u0 < nt * nh; u0 += kAppWarps * U) {
            Row r[U];
#pragma unroll
            for (int u = 0; u < U; u++)
                if (u0 + u < nt * nh) r[u].load(proj + (long)(t0 + (u0 + u) / nh) * a.proj_stride + a.q_off + (long)(h0 + (u0 + u) % nh) * a.d, a.d);
#pragma unroll
            for (int u = 0; u < U; u++)
                if (u0 + u < nt * nh) {
                    const int t = (u0 + u) / nh, h = h0 + (u0 + u) % nh;
                    r[u].prepare(proj + (long)(t0 + t) * a.proj_stride + a.q_off + (long)h * a.d, a, (const T*)a.q_w, [&](int i) { return table[t * half + i]; });
                    r[u].store((T*)a.q_out + ((long)(t0 + t) * a.H + h) * a.d, a.d);
                }
        }
        return;
    }
    const int g = blockIdx.x % a.G;
    if (warp == 0) {
        int s, item;
        const bool found = fp8_find(blockIdx.x / a.G, a.n_seqs, [&](int i) {
            const int start = a.seqs[i], len = a.seqs[a.seqs_stride + i];
            if (len <= 0 || start < 0 || start > a.n_tokens - len) return 0;
            const int p = a.pos[start];
            return p < 0 ? 0 : (p + len - 1) / ps - p / ps + 1;
        }, s, item);
        if (lane == 0) {
            info[0] = -1;
            if (found) {
                const int start = a.seqs[s], len = a.seqs[a.seqs_stride + s], p = a.pos[start], logical = p / ps + item;
                const int first = item ? logical * ps - p : 0, last = min(len, (logical + 1) * ps - p);      // the portion's tokens in this page
                info[0] = a.pages.page(a.slot[start], logical);
                info[1] = start + first;
                info[2] = last - first;
                info[3] = p + first;
            }
        }
    }
    __syncthreads();
    const int page = info[0], t0 = info[1], n = info[2], p0 = info[3], begun = p0 % ps;
    if (page < 0) return;
    const long block = (long)page * a.G + g;
    uint8_t *kc = a.k_codes + block * ps * a.d, *vc = a.v_codes + block * ps * a.dv;
    const int width = max(a.d, a.dv);
    const float old_k = begun ? a.scales[2 * block] : 0.f, old_v = begun ? a.scales[2 * block + 1] : 0.f;
    // rows 0 .. n - 1: keys, n .. 2 n - 1: values
    auto make = [&](Row& r, int u) {
        const bool is_v = u >= n;
        const int t = is_v ? u - n : u;
        const T* row = proj + (long)(t0 + t) * a.proj_stride + (is_v ? a.v_off + (long)g * a.dv : a.k_off + (long)g * a.d);
        r.load(row, is_v ? a.dv : a.d);
        if (!is_v) r.prepare(row, a, (const T*)a.k_w, [&](int i) { return app_turn(p0 + t, a.inv_freq[i]); });
    };
    float top_k = 0.f, top_v = 0.f;
    for (int u = warp; u < 2 * n; u += kAppWarps) {
        Row r;
        make(r, u);
        const float m = r.top(0);
        if (u >= n) top_v = fmaxf(top_v, m); else top_k = fmaxf(top_k, m);
        if (a.keep) {
#pragma unroll
            for (int e = 0; e < Row::N; e++)
                if (PER || Row::col(e) < width) app_smem[(long)u * width + Row::col(e)] = r.x[e];
        }
    }
    top_k = warp_max(top_k);
    top_v = warp_max(top_v);
    if (lane == 0) { tops[0][warp] = top_k; tops[1][warp] = top_v; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppWarps; w++) { top_k = fmaxf(top_k, tops[0][w]); top_v = fmaxf(top_v, tops[1][w]); }
    const float now_k = fmaxf(old_k, fp8_power(fp8_exponent(top_k))), now_v = fmaxf(old_v, fp8_power(fp8_exponent(top_v)));
    if (threadIdx.x == 0) { a.scales[2 * block] = now_k; a.scales[2 * block + 1] = now_v; }      // (every thread read the old ones ahead of the barrier)
    if (begun && now_k > old_k) fp8_move(kc, (long)begun * a.d, old_k / now_k);
    if (begun && now_v > old_v) fp8_move(vc, (long)begun * a.dv, old_v / now_v);
    const float inv_k = 1.0f / now_k, inv_v = 1.0f / now_v;
    for (int u = warp; u < 2 * n; u += kAppWarps) {
        Row r;
        if (a.keep) {
#pragma unroll
            for (int e = 0; e < Row::N; e++) r.x[e] = PER || Row::col(e) < width ? app_smem[(long)u * width + Row::col(e)] : 0.f;
        } else {
            make(r, u);
        }
        if (u >= n) r.store_codes(vc + (long)(begun + u - n) * a.dv, a.dv, inv_v);
        else r.store_codes(kc + (long)(begun + u) * a.d, a.d, inv_k);
    }
}

template <typename T, int PER> static cudaError_t launch_append(const Fp8Append& a, unsigned grid, size_t smem, cudaStream_t s) {
    const cudaError_t e = raise_smem_limit((const void*)fp8_append_kernel<T, PER>, smem);
    return e != cudaSuccess ? e : launch_pdl(fp8_append_kernel<T, PER>, dim3(grid), dim3(kAppThreads), smem, s, a);
}
template <typename T> static cudaError_t launch_append_of(const Fp8Append& a, int per, unsigned grid, size_t smem, cudaStream_t s) {
    return per == 2 ? launch_append<T, 2>(a, grid, smem, s) : per == 4 ? launch_append<T, 4>(a, grid, smem, s) : per == 8 ? launch_append<T, 8>(a, grid, smem, s) : launch_append<T, 0>(a, grid, smem, s);
}

}  // namespace ktb

using namespace ktb;

extern "C" int ktb200_fp8_cache_append(const ktb200_fp8_append_params* c, int n_tokens, int dtype, void* stream) {
    if (!c || c->heads <= 0 || c->kv_heads <= 0 || c->heads % c->kv_heads || c->dim <= 0 || c->dim > 32 * kAppCols || c->vdim <= 0 || c->vdim > 32 * kAppCols || c->rot_dims < 0 ||
        c->rot_dims > c->dim || (c->rot_dims & 1) || (c->rot_dims && !c->inv_freq) || (c->rot_layout != kRotInterleaved && c->rot_layout != kRotHalves) || c->page_size <= 0 ||
        c->max_pages <= 0 || c->n_pages < 0 || c->n_slots <= 0 || c->n_seqs < 0) {
        set_error("fp8_cache_append: bad argument (head sizes up to %d, an even number of turned columns)", 32 * kAppCols);
        return KTB200_EINVAL;
    }
    if (c->qk_norm != 0 && c->qk_norm != 1 && c->qk_norm != 3) { set_error("fp8_cache_append: qk_norm %d (0: none, 1: unit rms, 3: weighted ahead of the rotation)", c->qk_norm); return KTB200_EINVAL; }
    if (c->qk_norm == 3 && (!c->q_weight || !c->k_weight)) { set_error("fp8_cache_append: qk_norm 3 needs both weights"); return KTB200_EINVAL; }
    if (dtype != KTB200_TYPE_BF16 && dtype != KTB200_TYPE_F32) { set_error("fp8_cache_append: dtype must be bf16 or f32"); return KTB200_EINVAL; }
    if (n_tokens <= 0) return KTB200_OK;
    if (!c->proj || !c->pos || !c->slot || !c->seqs || !c->page_table || !c->k_codes || !c->v_codes || !c->scales || !c->q_out) { set_error("fp8_cache_append: null pointer"); return KTB200_EINVAL; }
    Fp8Append a{c->proj, c->proj_stride, c->q_off, c->k_off, c->v_off, c->heads, c->kv_heads, c->dim, c->vdim, c->rot_dims, c->rot_layout, c->inv_freq, c->qk_norm, c->q_weight, c->k_weight, c->eps,
                c->pos, c->slot, c->seqs, c->seqs_stride, c->n_seqs, n_tokens, {c->page_table, c->n_slots, c->max_pages, c->page_size, c->n_pages}, (uint8_t*)c->k_codes, (uint8_t*)c->v_codes,
                c->scales, c->q_out, 0, 0, 0, 0, 0};
    // a portion of n tokens meets n / page_size + 2 pages at most, and no more than n
    const long pages = c->n_seqs ? std::min<long>(n_tokens, n_tokens / c->page_size + 2L * c->n_seqs) : 0;
    // whole vectors of a lane's columns
    const size_t esz = dtype == KTB200_TYPE_BF16 ? 2 : 4;
    int per = c->dim == c->vdim && (c->dim == 64 || c->dim == 128 || c->dim == 256) ? c->dim / 32 : 0;
    if (per) {
        const size_t lane_bytes = std::min<size_t>(16, per * esz);
        auto whole = [&](const void* p) { return (reinterpret_cast<uintptr_t>(p) & (lane_bytes - 1)) == 0; };
        if (c->q_off % per || c->k_off % per || c->v_off % per || c->proj_stride % per || !whole(c->proj) || !whole(c->q_out) || (reinterpret_cast<uintptr_t>(c->k_codes) & (per - 1)) ||
            (reinterpret_cast<uintptr_t>(c->v_codes) & (per - 1)) || (c->rot_layout == kRotHalves ? (c->rot_dims / 2) % per : 0))
            per = 0;
    }
    // queries: a token's heads share its table of angles; eight units (one a warp) a CTA until the SMs are full, then four tokens with all their heads
    const bool many = (long)n_tokens * c->heads > 8 * 148 * 8;
    a.q_tokens = many ? 4 : 1;
    a.q_heads = many ? std::min(c->heads, 64) : std::min(c->heads, kAppWarps);
    a.q_blocks = (c->heads + a.q_heads - 1) / a.q_heads;
    const long q_ctas = ((long)n_tokens + a.q_tokens - 1) / a.q_tokens * a.q_blocks, kv_ctas = pages * c->kv_heads;
    if (q_ctas + kv_ctas > 0x7fffffffL) { set_error("fp8_cache_append: too many tokens"); return KTB200_EINVAL; }
    a.kv_ctas = (int)kv_ctas;
    // a page's rows stay in shared memory between the search for their largest and their codes where they fit
    const size_t rows = (size_t)2 * std::min(c->page_size, n_tokens) * std::max(c->dim, c->vdim) * sizeof(float);
    a.keep = rows <= kAppKeep;
    const size_t smem = std::max(a.keep ? rows : 0, (size_t)a.q_tokens * (c->rot_dims / 2) * sizeof(float2));
    KTB_CUDA_CHECK(dtype == KTB200_TYPE_BF16 ? launch_append_of<__nv_bfloat16>(a, per, (unsigned)(q_ctas + kv_ctas), smem, (cudaStream_t)stream)
                                             : launch_append_of<float>(a, per, (unsigned)(q_ctas + kv_ctas), smem, (cudaStream_t)stream));
    count_launch();
    return KTB200_OK;
}
