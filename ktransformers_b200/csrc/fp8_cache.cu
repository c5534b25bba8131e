// Appending keys and values to the paged e4m3 cache (fp8_cache.cuh), with the norms and the rotation applied on the way (libktb200_seq.so).
//
//   ktb200_fp8_cache_append   proj rows [... q ... k ... v ...]; q and k, head by head: nothing (qk_norm 0), x / sqrt(mean x^2 + eps) (1), the same times one weight per
//                             column (3); then a turn of the first rot_dims columns (pairs of either layout, angle pos * inv_freq[i]).  q to q_out; k and v as
//                             e4m3 codes under one scale per page and head.
//
// The tokens of a portion that fall into one page are appended by one CTA per key/value head for the keys and one for the values, which finds their largest magnitude, makes
// the block's scale, moves the codes of the tokens that the page held before where the scale has grown, and writes the new codes: no other CTA touches the block, so there
// is nothing to order and nothing to add up atomically.  A portion that begins at a page's first token starts its blocks anew (whatever the page held).
// Queries are turned and normed in fp32.  Keys are in fp64 up to their one rounding to fp32 ahead of the codes (the GPU does half as many fp64 operations as fp32 ones in a cycle, and a
// step's keys are few): their codes are those of the exact numbers, whatever the order of a sum.  Angles are fp64 in both.
#include <cuda_bf16.h>

#include <algorithm>

#include "fp8_cache.cuh"

namespace ktb {

constexpr int kAppCols = 8 /* columns of a lane: head sizes up to 256 */, kAppKeep = 48 * 1024 /* bytes of rows that a CTA keeps between the search for their largest and their codes */;

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
    int kv_ctas, q_heads, q_blocks, keep;      // CTAs of keys and values; query heads of a warp, warps of a token; rows of a page that fit in kAppKeep
};

template <typename F> struct AppTurn { F c, s; };
// (cos, sin) of pos * freq: the angle less a multiple of pi / 2, within pi / 4 of zero, and the first terms of both series (2e-14 and 1e-15 off)
template <typename F> __device__ __forceinline__ AppTurn<F> app_turn(int pos, double freq) {
    const double angle = (double)pos * freq, k = rint(angle * 0.63661977236758134), r = fma(-k, 6.123233995736766e-17, fma(-k, 1.5707963267948966, angle)), x = r * r;
    double s = fma(x, 1.0 / 6227020800.0, -1.0 / 39916800.0), c = fma(x, -1.0 / 87178291200.0, 1.0 / 479001600.0);
    s = fma(x, s, 1.0 / 362880.0);
    c = fma(x, c, -1.0 / 3628800.0);
    s = fma(x, s, -1.0 / 5040.0);
    c = fma(x, c, 1.0 / 40320.0);
    s = fma(x, s, 1.0 / 120.0);
    c = fma(x, c, -1.0 / 720.0);
    s = fma(x, s, -1.0 / 6.0);
    c = fma(x, c, 1.0 / 24.0);
    s = fma(r * x, s, r);
    c = fma(x, fma(x, c, -0.5), 1.0);
    const int quarter = (int)k;
    const double u = quarter & 1 ? s : c, v = quarter & 1 ? c : s;      // cos and sin of the angle but for their signs
    return {(F)((quarter + 1) & 2 ? -u : u), (F)(quarter & 2 ? -v : v)};
}
template <typename F> __device__ __forceinline__ F app_sum(F v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float app_inv_root(float x) { return rsqrtf(x); }      // (2 ulp; a correctly rounded root and quotient are 20 instructions a row)
__device__ __forceinline__ double app_inv_root(double x) { return rsqrt(x); }

// One head's columns of one token, as a warp holds them.  PER > 0: heads of 32 PER columns, a lane's PER of them side by side; PER = 0: any size, columns lane, lane + 32, ..
template <typename T, int PER, bool HALVES> struct AppRow {
    static constexpr int N = PER ? PER : kAppCols;
    float x[N];
    __device__ __forceinline__ static int col(int e) { const int lane = threadIdx.x & 31; return PER ? lane * PER + e : lane + 32 * e; }
    static constexpr int W = PER ? PER * (int)sizeof(T) / 4 : 1;      // words of a lane's columns as they are stored
    __device__ __forceinline__ static void fetch(uint32_t (&w)[W], const T* row) {
        const void* from = row + col(0);
        if constexpr (W == 1) w[0] = *reinterpret_cast<const uint32_t*>(from);
        else if constexpr (W == 2) { const uint2 v = *reinterpret_cast<const uint2*>(from); w[0] = v.x; w[1] = v.y; }
        else {
#pragma unroll
            for (int i = 0; i < W; i += 4) { const uint4 v = reinterpret_cast<const uint4*>(from)[i / 4]; w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w; }
        }
    }
    __device__ __forceinline__ void unpack(const uint32_t (&w)[W]) {
#pragma unroll
        for (int i = 0; i < W; i++) {
            if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w[i]);
            else { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
        }
    }
    // a lane's columns on their way to shared memory (the lane reads them there itself)
    __device__ __forceinline__ static void bring(T* to, const T* row) {
        constexpr int B = W * 4 < 16 ? W * 4 : 16;
        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to + col(0));
        const char* src = reinterpret_cast<const char*>(row + col(0));
#pragma unroll
        for (int i = 0; i < W * 4; i += B) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst + i), "l"(src + i), "n"(B) : "memory");
    }
    __device__ __forceinline__ void load(const T* row, int n) {
        if constexpr (PER == 0) {
#pragma unroll
            for (int e = 0; e < N; e++) x[e] = col(e) < n ? to_f(row[col(e)]) : 0.f;
        } else {
            uint32_t w[W];
            fetch(w, row);
            unpack(w);
        }
    }
    // The turns of a lane's columns at a position.  Two columns share each: two neighbours of a lane, or (halves) one of this lane and one of its partner, of which each makes half
    template <typename F> __device__ __forceinline__ static void turns(const Fp8Append& a, int pos, AppTurn<F> (&t)[N]) {
        const int half = a.rot_dims >> 1, lane = threadIdx.x & 31;
        if constexpr (PER == 0) {
#pragma unroll
            for (int e = 0; e < N; e++) {
                const int c = col(e);
                t[e] = {F(1), F(0)};
                if (c < a.rot_dims) t[e] = app_turn<F>(pos, a.inv_freq[a.rot_layout == kRotHalves ? (c >= half ? c - half : c) : c >> 1]);
            }
        } else if constexpr (!HALVES) {
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                const int c = col(e);
                t[e] = {F(1), F(0)};
                if (c < a.rot_dims) t[e] = app_turn<F>(pos, a.inv_freq[c >> 1]);
                t[e + 1] = t[e];
            }
        } else {
            const int step = half / (PER ? PER : 1);
            const bool second = col(0) >= half, in = col(0) < a.rot_dims;
            const int partner = second ? lane - step : lane + step;
#pragma unroll
            for (int e = 0; e < N / 2; e++) {
                AppTurn<F> own{F(1), F(0)};
                if (in) own = app_turn<F>(pos, a.inv_freq[col(second ? e + N / 2 : e) - (second ? half : 0)]);
                const AppTurn<F> other{__shfl_sync(0xffffffffu, own.c, partner), __shfl_sync(0xffffffffu, own.s, partner)};
                t[e] = second && in ? other : own;
                t[e + N / 2] = second && in ? own : other;
            }
            if (!in) {
#pragma unroll
                for (int e = 0; e < N; e++) t[e] = {F(1), F(0)};
            }
        }
    }
    // the weights of a lane's columns (qk_norm 3; one elsewhere)
    __device__ __forceinline__ static void weights(const Fp8Append& a, const T* w, float (&to)[N]) {
#pragma unroll
        for (int e = 0; e < N; e++) to[e] = a.qk_norm == 3 && (PER || col(e) < a.d) ? to_f(w[col(e)]) : 1.f;
    }
    // norm and turn, in F, then back to fp32 (row, w: what PER = 0 reads its partners from)
    template <typename F> __device__ __forceinline__ void prepare(const T* row, const Fp8Append& a, const T* w, const float (&wv)[N], const AppTurn<F> (&t)[N]) {
        const int lane = threadIdx.x & 31, half = a.rot_dims >> 1;
        F y[N], inv = F(1);
#pragma unroll
        for (int e = 0; e < N; e++) y[e] = (F)x[e];
        if (a.qk_norm) {
            F ss = F(0);
#pragma unroll
            for (int e = 0; e < N; e++) ss = fma(y[e], y[e], ss);
            inv = app_inv_root(app_sum(ss) / (F)a.d + (F)a.eps);
#pragma unroll
            for (int e = 0; e < N; e++) y[e] = y[e] * inv * (F)wv[e];
        }
        if constexpr (PER > 0 && !HALVES) {
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                const F u = y[e], v = y[e + 1];
                y[e] = u * t[e].c - v * t[e].s;
                y[e + 1] = v * t[e].c + u * t[e].s;
            }
        } else if constexpr (PER > 0) {      // halves: the partner's lane is half / PER lanes away; the signs of the sines are in s (columns that do not turn: 0)
            const int step = half / PER, c = col(0), partner = c >= half ? lane - step : lane + step;
            const F sign = c >= half ? F(1) : F(-1);
#pragma unroll
            for (int e = 0; e < N; e++) {
                const F other = __shfl_sync(0xffffffffu, y[e], partner);
                y[e] = y[e] * t[e].c + other * (sign * t[e].s);
            }
        } else if (a.rot_dims) {
#pragma unroll
            for (int e = 0; e < N; e++) {
                const int c = col(e);
                if (c < a.rot_dims) {
                    const int o = rot_partner(c, a.rot_dims, a.rot_layout);
                    const bool second = a.rot_layout == kRotHalves ? c >= half : (c & 1);
                    F other = (F)to_f(row[o]) * inv;
                    if (a.qk_norm == 3) other *= (F)to_f(w[o]);
                    y[e] = second ? y[e] * t[e].c + other * t[e].s : y[e] * t[e].c - other * t[e].s;
                }
            }
        }
#pragma unroll
        for (int e = 0; e < N; e++) x[e] = (float)y[e];
    }
    __device__ __forceinline__ float top() const {
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
        for (long i = 4 * (long)threadIdx.x; i < bytes; i += 4 * blockDim.x) {
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
        for (long i = threadIdx.x; i < bytes; i += blockDim.x) {
            const float x = __half2float(__half(__nv_cvt_fp8_to_halfraw(p[i], __NV_E4M3)));
            p[i] = (uint8_t)__nv_cvt_float_to_fp8(x * f, __NV_SATFINITE, __NV_E4M3);
        }
    }
}

// Blocks [0, kv_ctas): the keys or the values of one page's tokens of one portion for one key/value head (the portions' pages in order, then heads, keys ahead of values); the
// blocks behind them: a warp has q_heads query heads of one token, whose turns it makes once.
// Bound by the bytes of proj, q and the codes: what counts is rows in flight, eight a warp of queries, a CTA's whole page of keys or values.
template <typename T, int PER, bool HALVES> __global__ void __launch_bounds__(256, PER == 8 || PER == 0 ? 2 : 3) fp8_append_kernel(const Fp8Append a) {
    using Row = AppRow<T, PER, HALVES>;
    extern __shared__ __align__(16) unsigned char app_smem[];
    __shared__ float tops[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5, ps = a.pages.page_size;
    const T* proj = (const T*)a.proj;
    griddep_launch_dependents();
    griddep_wait();
    if ((int)blockIdx.x >= a.kv_ctas) {
        const long unit = (long)(blockIdx.x - a.kv_ctas) * nw + warp;
        const int t = (int)(unit / a.q_blocks), h0 = (int)(unit % a.q_blocks) * a.q_heads, h1 = min(a.H, h0 + a.q_heads);
        if (t >= a.n_tokens) return;
        const T* row = proj + (long)t * a.proj_stride + a.q_off;
        T* out = (T*)a.q_out + (long)t * a.H * a.d;
        row += (long)h0 * a.d;
        out += (long)h0 * a.d;
        int left = h1 - h0;
        AppTurn<float> turn[Row::N];
        float wv[Row::N];
        constexpr int U = PER == 0 ? 1 : Row::W <= 4 ? 8 : 4;
        uint32_t w[U][Row::W];
        if constexpr (PER > 0) {
            if (left >= U) {
#pragma unroll
                for (int u = 0; u < U; u++) Row::fetch(w[u], row + u * a.d);
            }
        }
        Row::turns(a, a.pos[t], turn);
        Row::weights(a, (const T*)a.q_w, wv);
        if constexpr (PER > 0) {
            while (left >= U) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    Row r;
                    r.unpack(w[u]);
                    if (left >= U + U) Row::fetch(w[u], row + (U + u) * a.d);
                    r.prepare(row, a, (const T*)a.q_w, wv, turn);
                    r.store(out + u * a.d, a.d);
                }
                left -= U;
                row += U * a.d;
                out += U * a.d;
            }
        }
        for (; left > 0; left--, row += a.d, out += a.d) {
            Row r;
            r.load(row, a.d);
            r.prepare(row, a, (const T*)a.q_w, wv, turn);
            r.store(out, a.d);
        }
        return;
    }
    const bool is_v = blockIdx.x & 1;
    const int g = (blockIdx.x >> 1) % a.G;
    int s, item, start = 0, len = 0, pos = 0, slot = 0;
    const bool found = fp8_find((blockIdx.x >> 1) / a.G, a.n_seqs, [&](int i) {
        start = a.seqs[i];
        len = a.seqs[a.seqs_stride + i];
        if (len <= 0 || start < 0 || start > a.n_tokens - len) return 0;
        pos = a.pos[start];
        slot = a.slot[start];
        return pos < 0 ? 0 : (pos + len - 1) / ps - pos / ps + 1;
    }, s, item);
    if (!found) return;
    start = __shfl_sync(0xffffffffu, start, s & 31);
    len = __shfl_sync(0xffffffffu, len, s & 31);
    pos = __shfl_sync(0xffffffffu, pos, s & 31);
    slot = __shfl_sync(0xffffffffu, slot, s & 31);
    const int logical = pos / ps + item, first = item ? logical * ps - pos : 0, n = min(len, (logical + 1) * ps - pos) - first;      // the portion's tokens in this page
    const int t0 = start + first, p0 = pos + first, begun = p0 % ps, page = a.pages.page(slot, logical), width = is_v ? a.dv : a.d;
    const T* rows = proj + (long)t0 * a.proj_stride + (is_v ? a.v_off + (long)g * a.dv : a.k_off + (long)g * a.d);
    // A warp has rows warp, warp + nw, ..: of a.keep at a time the columns as they came (PER > 0) and, of keys that were turned or normed, the results
    T* raw = reinterpret_cast<T*>(app_smem);
    float* done = reinterpret_cast<float*>(app_smem + (PER ? (size_t)a.keep * max(a.d, a.dv) * sizeof(T) : 0));
    const bool work = !is_v && (a.rot_dims || a.qk_norm), kept = n <= a.keep;
    float top = 0.f, wv[Row::N];
    if (work) Row::weights(a, (const T*)a.k_w, wv);
    auto make = [&](int base) {
        const int end = min(n, base + a.keep);
        if constexpr (PER > 0) {
            for (int t = base + warp; t < end; t += nw) Row::bring(raw + (long)(t - base) * width, rows + (long)t * a.proj_stride);
            asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
        }
#pragma unroll 1
        for (int t = base + warp; t < end; t += nw) {
            Row r;
            const T* row = rows + (long)t * a.proj_stride;
            r.load(PER ? raw + (long)(t - base) * width : row, width);
            if (work) {
                AppTurn<double> turn[Row::N];
                Row::turns(a, p0 + t, turn);
                r.prepare(row, a, (const T*)a.k_w, wv, turn);
            }
            if (work || PER == 0) {
#pragma unroll
                for (int e = 0; e < Row::N; e++)
                    if (PER || Row::col(e) < width) done[(long)(t - base) * width + Row::col(e)] = r.x[e];
            }
            top = fmaxf(top, r.top());
        }
    };
    auto codes_of = [&](int base, uint8_t* codes, float inv) {
        const int end = min(n, base + a.keep);
        for (int t = base + warp; t < end; t += nw) {
            Row r;
            if (work || PER == 0) {
#pragma unroll
                for (int e = 0; e < Row::N; e++) r.x[e] = PER || Row::col(e) < width ? done[(long)(t - base) * width + Row::col(e)] : 0.f;
            } else {
                r.load(raw + (long)(t - base) * width, width);
            }
            r.store_codes(codes + (long)(begun + t) * width, width, inv);
        }
    };
    for (int base = 0; base < n; base += a.keep) make(base);
    if (page < 0) return;
    const long block = (long)page * a.G + g;
    uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + block * ps * width;
    float* scale = a.scales + 2 * block + is_v;
    const float old = begun ? *scale : 0.f;
    top = warp_max(top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    for (int w = 0; w < nw; w++) top = fmaxf(top, tops[w]);
    const float now = fmaxf(old, fp8_power(fp8_exponent(top))), inv = 1.0f / now;
    if (threadIdx.x == 0) *scale = now;      // (every thread read the old one ahead of the barrier)
    if (begun && now > old) fp8_move(codes, (long)begun * width, old / now);
    if (kept) {
        codes_of(0, codes, inv);
    } else {
        for (int base = 0; base < n; base += a.keep) {      // (more rows than the CTA keeps: once more)
            make(base);
            codes_of(base, codes, inv);
        }
    }
}

template <typename T> static cudaError_t launch_append(const Fp8Append& a, int per, unsigned grid, int threads, size_t smem, cudaStream_t s) {
    const bool halves = a.rot_layout == kRotHalves;
    const auto kernel = per == 2   ? (halves ? fp8_append_kernel<T, 2, true> : fp8_append_kernel<T, 2, false>)
                        : per == 4 ? (halves ? fp8_append_kernel<T, 4, true> : fp8_append_kernel<T, 4, false>)
                        : per == 8 ? (halves ? fp8_append_kernel<T, 8, true> : fp8_append_kernel<T, 8, false>)
                                   : fp8_append_kernel<T, 0, false>;
    const cudaError_t e = raise_smem_limit((const void*)kernel, smem);
    return e != cudaSuccess ? e : launch_pdl(kernel, dim3(grid), dim3(threads), smem, s, a);
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
                c->scales, c->q_out, 0, 0, 0, 0};
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
    // decode steps bring one row to most blocks: two warps a CTA; prompts eight
    const int threads = (long)n_tokens <= 4L * c->n_seqs ? 64 : 256, nw = threads / 32;
    // query heads of a warp: as many as leave about 32 warps an SM
    a.q_heads = (int)std::max<long>(1, std::min<long>({32, c->heads, (long)n_tokens * c->heads / (148 * 32)}));
    a.q_blocks = (c->heads + a.q_heads - 1) / a.q_heads;
    const long q_ctas = ((long)n_tokens * a.q_blocks + nw - 1) / nw, kv_ctas = 2 * pages * c->kv_heads;
    if (q_ctas + kv_ctas > 0x7fffffffL) { set_error("fp8_cache_append: too many tokens"); return KTB200_EINVAL; }
    a.kv_ctas = (int)kv_ctas;
    const size_t row_bytes = (size_t)std::max(c->dim, c->vdim) * ((per ? esz : 0) + sizeof(float));
    a.keep = (int)std::min<size_t>(threads == 64 ? 8 : std::min(c->page_size, n_tokens), kAppKeep / row_bytes);      // (decode: little shared memory, many CTAs)
    const size_t smem = a.keep * row_bytes;
    KTB_CUDA_CHECK(dtype == KTB200_TYPE_BF16 ? launch_append<__nv_bfloat16>(a, per, (unsigned)(q_ctas + kv_ctas), threads, smem, (cudaStream_t)stream)
                                             : launch_append<float>(a, per, (unsigned)(q_ctas + kv_ctas), threads, smem, (cudaStream_t)stream));
    count_launch();
    return KTB200_OK;
}
