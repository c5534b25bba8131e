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
template <int LANES, typename F> __device__ __forceinline__ F app_sum(F v) {      // over groups of LANES lanes
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float app_inv_root(float x) { return rsqrtf(x); }      // (2 ulp; a correctly rounded root and quotient are 20 instructions a row)
__device__ __forceinline__ double app_inv_root(double x) { return rsqrt(x); }

// One head's columns of one token: LPR lanes have eight each (head sizes 64, 128 and 256), so that a warp has 32 / LPR rows at a time; LPR = 0: any size, the whole warp one row, columns
// lane, lane + 32, ..  A lane's eight are two runs of four at c0 and c1.  HALVES: a turned lane's runs are rot_dims / 2 apart, so that pairs meet in a lane; every other lane's are
// side by side.
template <typename T, int LPR, bool HALVES> struct AppRow {
    static constexpr int N = kAppCols, PAIRS = LPR ? 4 : N, LANES = LPR ? LPR : 32, ROWS = 32 / LANES, W = LPR ? (int)sizeof(T) : 1;      // W: words of four columns, twice
    float x[N];
    struct Place { int c0, c1, pair; };      // pair: the first of a lane's four (neighbours or halves), or -1: not turned
    __device__ __forceinline__ static Place place(const Fp8Append& a, int lane_in_row, bool turned) {
        const int r = turned ? a.rot_dims : 0;
        if (HALVES && 8 * lane_in_row < r) return {4 * lane_in_row, r / 2 + 4 * lane_in_row, 4 * lane_in_row};
        return {8 * lane_in_row, 8 * lane_in_row + 4, 8 * lane_in_row < r ? 4 * lane_in_row : -1};
    }
    __device__ __forceinline__ static int col(int e) { return (threadIdx.x & 31) + 32 * e; }      // (LPR = 0)
    __device__ __forceinline__ static void fetch(uint32_t (&w)[2 * W], const T* row, const Place& p) {
        if constexpr (W == 2) {
            const uint2 u = *reinterpret_cast<const uint2*>(row + p.c0), v = *reinterpret_cast<const uint2*>(row + p.c1);
            w[0] = u.x; w[1] = u.y; w[2] = v.x; w[3] = v.y;
        } else if constexpr (W == 4) {
            const uint4 u = *reinterpret_cast<const uint4*>(row + p.c0), v = *reinterpret_cast<const uint4*>(row + p.c1);
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w; w[4] = v.x; w[5] = v.y; w[6] = v.z; w[7] = v.w;
        }
    }
    __device__ __forceinline__ void unpack(const uint32_t (&w)[2 * W]) {
        if constexpr (LPR > 0) {
#pragma unroll
            for (int i = 0; i < 2 * W; i++) {
                if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w[i]);
                else { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
            }
        }
    }
    // a lane's columns on their way to shared memory (the lane reads them there itself)
    __device__ __forceinline__ static void bring(T* to, const T* row, const Place& p) {
        constexpr int B = 4 * sizeof(T);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int c = i ? p.c1 : p.c0;
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to + c)), "l"(row + c), "n"(B) : "memory");
        }
    }
    __device__ __forceinline__ void load(const T* row, int n, const Place& p) {
        if constexpr (LPR == 0) {
#pragma unroll
            for (int e = 0; e < N; e++) x[e] = col(e) < n ? to_f(row[col(e)]) : 0.f;
        } else {
            uint32_t w[2 * W];
            fetch(w, row, p);
            unpack(w);
        }
    }
    // the turns of a lane's pairs (LPR = 0: of its columns) at a position
    template <typename F> __device__ __forceinline__ static void turns(const Fp8Append& a, int pos, const Place& p, AppTurn<F> (&t)[PAIRS]) {
        const int half = a.rot_dims >> 1;
#pragma unroll
        for (int e = 0; e < PAIRS; e++) {
            t[e] = {F(1), F(0)};
            if constexpr (LPR > 0) {
                if (p.pair >= 0) t[e] = app_turn<F>(pos, a.inv_freq[p.pair + e]);
            } else {
                const int c = col(e);
                if (c < a.rot_dims) t[e] = app_turn<F>(pos, a.inv_freq[a.rot_layout == kRotHalves ? (c >= half ? c - half : c) : c >> 1]);
            }
        }
    }
    // the weights of a lane's columns (qk_norm 3; one elsewhere)
    __device__ __forceinline__ static void weights(const Fp8Append& a, const T* w, const Place& p, float (&to)[N]) {
#pragma unroll
        for (int e = 0; e < N; e++) {
            const int c = LPR ? (e < 4 ? p.c0 + e : p.c1 + e - 4) : col(e);
            to[e] = a.qk_norm == 3 && c < a.d ? to_f(w[c]) : 1.f;
        }
    }
    // norm and turn, in F, then back to fp32 (row, w: what LPR = 0 reads its partners from)
    template <typename F> __device__ __forceinline__ void prepare(const T* row, const Fp8Append& a, const T* w, const float (&wv)[N], const AppTurn<F> (&t)[PAIRS]) {
        F y[N], inv = F(1);
#pragma unroll
        for (int e = 0; e < N; e++) y[e] = (F)x[e];
        if (a.qk_norm) {
            F ss = F(0);
#pragma unroll
            for (int e = 0; e < N; e++) ss = fma(y[e], y[e], ss);
            inv = app_inv_root(app_sum<LANES>(ss) / (F)a.d + (F)a.eps);
#pragma unroll
            for (int e = 0; e < N; e++) y[e] = y[e] * inv * (F)wv[e];
        }
        if constexpr (LPR > 0) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = HALVES ? i : 2 * i, o = HALVES ? i + 4 : 2 * i + 1;
                const F u = y[e], v = y[o];
                y[e] = u * t[i].c - v * t[i].s;
                y[o] = v * t[i].c + u * t[i].s;
            }
        } else if (a.rot_dims) {
            const int half = a.rot_dims >> 1;
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
    template <typename D> __device__ __forceinline__ void store(D* row, int n, const Place& p) const {
        if constexpr (LPR == 0) {
#pragma unroll
            for (int e = 0; e < N; e++)
                if (col(e) < n) row[col(e)] = from_f<D>(x[e]);
        } else {
            store4(row + p.c0, make_float4(x[0], x[1], x[2], x[3]));
            store4(row + p.c1, make_float4(x[4], x[5], x[6], x[7]));
        }
    }
    __device__ __forceinline__ void load_done(const float* row, int n, const Place& p) {
        if constexpr (LPR == 0) {
#pragma unroll
            for (int e = 0; e < N; e++) x[e] = col(e) < n ? row[col(e)] : 0.f;
        } else {
            const float4 u = load4(row + p.c0), v = load4(row + p.c1);
            x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
        }
    }
    __device__ __forceinline__ void store_codes(uint8_t* row, int n, float inv_scale, const Place& p) const {
        if constexpr (LPR == 0) {
#pragma unroll
            for (int e = 0; e < N; e++)
                if (col(e) < n) row[col(e)] = (uint8_t)__nv_cvt_float_to_fp8(x[e] * inv_scale, __NV_SATFINITE, __NV_E4M3);
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i] * inv_scale, x[4 * i + 1] * inv_scale), __NV_SATFINITE, __NV_E4M3);
                const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2] * inv_scale, x[4 * i + 3] * inv_scale), __NV_SATFINITE, __NV_E4M3);
                *reinterpret_cast<uint32_t*>(row + (i ? p.c1 : p.c0)) = lo | hi << 16;
            }
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
// Bound by the bytes of proj, q and the codes: what counts is rows in flight, and instructions a row: two rows of 128 columns a warp and no exchange between lanes but for a norm's sum.
template <typename T, int LPR, bool HALVES> __global__ void __launch_bounds__(256, LPR == 0 ? 2 : 3) fp8_append_kernel(const Fp8Append a) {
    using Row = AppRow<T, LPR, HALVES>;
    extern __shared__ __align__(16) unsigned char app_smem[];
    __shared__ float tops[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5, ps = a.pages.page_size, sub = lane / Row::LANES, in_row = lane % Row::LANES;
    const T* proj = (const T*)a.proj;
    griddep_launch_dependents();
    griddep_wait();
    if ((int)blockIdx.x >= a.kv_ctas) {
        const long unit = (long)(blockIdx.x - a.kv_ctas) * nw + warp;
        const int t = (int)(unit / a.q_blocks), h0 = (int)(unit % a.q_blocks) * a.q_heads, n = min(a.H - h0, a.q_heads);
        if (t >= a.n_tokens) return;
        const typename Row::Place p = Row::place(a, in_row, true);
        const T* row = proj + (long)t * a.proj_stride + a.q_off + (long)h0 * a.d;
        T* out = (T*)a.q_out + ((long)t * a.H + h0) * a.d;
        AppTurn<float> turn[Row::PAIRS];
        float wv[Row::N];
        constexpr int U = LPR == 0 ? 1 : 4, STEP = U * Row::ROWS;      // U groups of a warp's rows on their way at once
        uint32_t w[U][2 * Row::W];
        int h = 0;
        if constexpr (LPR > 0) {
            if (STEP <= n) {
#pragma unroll
                for (int u = 0; u < U; u++) Row::fetch(w[u], row + (long)(u * Row::ROWS + sub) * a.d, p);
            }
        }
        Row::turns(a, a.pos[t], p, turn);
        Row::weights(a, (const T*)a.q_w, p, wv);
        if constexpr (LPR > 0) {
            for (; h + STEP <= n; h += STEP) {
                const bool more = h + 2 * STEP <= n;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const long at = (long)(h + u * Row::ROWS + sub) * a.d;
                    Row r;
                    r.unpack(w[u]);
                    if (more) Row::fetch(w[u], row + at + (long)STEP * a.d, p);
                    r.prepare(row, a, (const T*)a.q_w, wv, turn);
                    r.store(out + at, a.d, p);
                }
            }
        }
        for (; h < n; h += Row::ROWS) {
            const bool mine = h + sub < n;
            const long at = (long)(mine ? h + sub : h) * a.d;
            Row r;
            r.load(row + at, a.d, p);
            r.prepare(row + at, a, (const T*)a.q_w, wv, turn);
            if (mine) r.store(out + at, a.d, p);
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
    const int logical = pos / ps + item;
    if ((pos + len - 1) / ps - logical >= a.pages.max_pages) return;      // the portion itself goes once round the ring and writes the page again
    const int first = item ? logical * ps - pos : 0, n = min(len, (logical + 1) * ps - pos) - first;      // the portion's tokens in this page
    const int t0 = start + first, p0 = pos + first, begun = p0 % ps, page = a.pages.page(slot, logical), width = is_v ? a.dv : a.d;
    const T* rows = proj + (long)t0 * a.proj_stride + (is_v ? a.v_off + (long)g * a.dv : a.k_off + (long)g * a.d);
    // A warp has groups of its rows, nw groups apart: of a.keep rows at a time the columns as they came (LPR > 0) and, of keys that were turned or normed, the results
    const bool work = !is_v && (a.rot_dims || a.qk_norm), kept = n <= a.keep;
    const typename Row::Place place = Row::place(a, in_row, work);
    T* raw = reinterpret_cast<T*>(app_smem);
    float* done = reinterpret_cast<float*>(app_smem + (LPR ? (size_t)a.keep * a.d * sizeof(T) : 0));
    float top = 0.f, wv[Row::N];
    if (work) Row::weights(a, (const T*)a.k_w, place, wv);
    auto make = [&](int base) {
        const int end = min(n, base + a.keep);
        __syncwarp();      // (of the pass before, all lanes have read the columns)
        if constexpr (LPR > 0) {
            for (int t = base + warp * Row::ROWS + sub; t < end; t += nw * Row::ROWS) Row::bring(raw + (long)(t - base) * width, rows + (long)t * a.proj_stride, place);
            asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
        }
#pragma unroll 1
        for (int t0 = base + warp * Row::ROWS; t0 < end; t0 += nw * Row::ROWS) {
            const bool mine = t0 + sub < end;
            const int t = mine ? t0 + sub : t0;      // (a row that is not there: the group's first once more, whose columns another lane brought)
            __syncwarp();
            Row r;
            const T* row = rows + (long)t * a.proj_stride;
            r.load(LPR ? raw + (long)(t - base) * width : row, width, place);
            if (work) {
                AppTurn<double> turn[Row::PAIRS];
                Row::turns(a, p0 + t, place, turn);
                r.prepare(row, a, (const T*)a.k_w, wv, turn);
            }
            if ((work || LPR == 0) && mine) r.store(done + (long)(t - base) * width, width, place);
            top = fmaxf(top, r.top());
        }
    };
    auto codes_of = [&](int base, uint8_t* codes, float inv) {
        const int end = min(n, base + a.keep);
        for (int t = base + warp * Row::ROWS + sub; t < end; t += nw * Row::ROWS) {
            Row r;
            if (work || LPR == 0) r.load_done(done + (long)(t - base) * width, width, place);
            else r.load(raw + (long)(t - base) * width, width, place);
            r.store_codes(codes + (long)(begun + t) * width, width, inv, place);
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

template <typename T> static cudaError_t launch_append(const Fp8Append& a, int lanes, unsigned grid, int threads, size_t smem, cudaStream_t s) {
    const bool halves = a.rot_layout == kRotHalves;
    const auto kernel = lanes == 8    ? (halves ? fp8_append_kernel<T, 8, true> : fp8_append_kernel<T, 8, false>)
                        : lanes == 16 ? (halves ? fp8_append_kernel<T, 16, true> : fp8_append_kernel<T, 16, false>)
                        : lanes == 32 ? (halves ? fp8_append_kernel<T, 32, true> : fp8_append_kernel<T, 32, false>)
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
    // eight columns a lane, four at a time
    const size_t esz = dtype == KTB200_TYPE_BF16 ? 2 : 4;
    int lanes = c->dim == c->vdim && (c->dim == 64 || c->dim == 128 || c->dim == 256) && c->rot_dims % 8 == 0 ? c->dim / 8 : 0;
    if (lanes) {
        auto whole = [&](const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; };
        if (c->q_off % 4 || c->k_off % 4 || c->v_off % 4 || c->proj_stride % 4 || !whole(c->proj, 4 * esz) || !whole(c->q_out, 4 * esz) || !whole(c->k_codes, 4) || !whole(c->v_codes, 4)) lanes = 0;
    }
    // decode steps bring one row to most blocks: two warps a CTA; prompts eight
    const int threads = (long)n_tokens <= 4L * c->n_seqs ? 64 : 256, nw = threads / 32;
    // query heads of a warp: as many as leave about 32 warps an SM, whole groups of its rows
    const long group = lanes ? 32 / lanes : 1, want = (long)n_tokens * c->heads / (148 * 32);
    a.q_heads = (int)std::min<long>(32, std::max(group, want / group * group));
    a.q_blocks = (c->heads + a.q_heads - 1) / a.q_heads;
    const long q_ctas = ((long)n_tokens * a.q_blocks + nw - 1) / nw, kv_ctas = 2 * pages * c->kv_heads;
    if (q_ctas + kv_ctas > 0x7fffffffL) { set_error("fp8_cache_append: too many tokens"); return KTB200_EINVAL; }
    a.kv_ctas = (int)kv_ctas;
    const size_t row_bytes = (size_t)std::max(c->dim, c->vdim) * ((lanes ? esz : 0) + sizeof(float));
    a.keep = (int)std::min<size_t>(threads == 64 ? 8 : std::min(c->page_size, n_tokens), kAppKeep / row_bytes);      // (decode: little shared memory, many CTAs)
    const size_t smem = a.keep * row_bytes;
    KTB_CUDA_CHECK(dtype == KTB200_TYPE_BF16 ? launch_append<__nv_bfloat16>(a, lanes, (unsigned)(q_ctas + kv_ctas), threads, smem, (cudaStream_t)stream)
                                             : launch_append<float>(a, lanes, (unsigned)(q_ctas + kv_ctas), threads, smem, (cudaStream_t)stream));
    count_launch();
    return KTB200_OK;
}
