// Soft-max attention over grouped key/value heads in the paged e4m3 cache of fp8_cache.cuh (libktb200_seq.so).
//
//   ktb200_fp8_cache_attn   o_i = sum_j w_ij v_j / sum_j w_ij over the keys j <= i with i - j < window (window > 0) and floor(j / chunk) == floor(i / chunk) (chunk > 0);
//                           w_ij = exp(s_ij), s_ij = cap(scale t_h q_i.k_j), cap(s) = c tanh(s / c), c = softcap (softcap <= 0: none), t_h a number per query head
//                           (optional); exp(sink_h) joins the denominator (optional); o times out_scale.  k_j, v_j: codes times their blocks' scales.  Query head h reads
//                           key/value head h / (H / G).  The key range is cut into splits for few tokens on long ranges.
//
// A portion's tokens stand at consecutive positions from pos[its first token].  Keys in pages that are not there (ids outside the pool) are not seen; a row that sees no key
// becomes zero.  Rows of tokens that belong to no portion are left as they were.
#include <cuda_bf16.h>

#include <algorithm>

#include "fp8_cache.cuh"

namespace ktb {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kFp8MaxParts = 128, kFp8MinPart = 256, kFp8MaxDim = 256;

struct Fp8Attn {
    const void* q;
    int H, G, d, dv;
    float scale;
    const float* head_scale;
    float softcap;
    int window, chunk;
    const float* sink;
    float out_scale;
    const int *pos, *slot, *seqs;
    int seqs_stride, n_seqs, n_tokens;
    Fp8Pages pages;
    const uint8_t *k_codes, *v_codes;
    const float* scales;
    void* out;
    long out_stride;
    float* partial;      // [T][H][parts][dv + 2]: reference maximum, sum, un-normalised weighted values
    int part, parts;     // keys of a part (0: the range is not cut), and the most parts of a range
    int even;            // or: into so many parts of about the same length, one cluster's (0: not)
    int ctoks, align;    // tokens of a CTA: their range, from the first visible key of the first of them (rounded down to align) on, is what is cut
};
__device__ __forceinline__ int fp8_first_visible(int p, int window, int chunk) {
    int lo = window > 0 ? max(0, p - window + 1) : 0;
    if (chunk > 0) lo = max(lo, p - p % chunk);
    return lo;
}
// The sink's term in a row's sum l over the reference m (both, and the sink, as exponents of two); returns what the row's other sums are multiplied by.  An infinite sink takes all (+) or
// nothing (-), and a row that sees no key stays at zero beside either
__device__ __forceinline__ float fp8_sink(float sink, float m, float& l) {
    const float sk = sink * kLog2e, mn = fmaxf(m, sk), k = m == -INFINITY ? 0.f : exp2_approx(m - mn);
    l = l * k + (sk == mn ? 1.f : exp2_approx(sk - mn));
    return k;
}
// tokens of portion s (none where its rows are not those of the step)
__device__ __forceinline__ int fp8_portion(const Fp8Attn& a, int s) {
    const int start = a.seqs[s], len = a.seqs[a.seqs_stride + s];
    return len <= 0 || start < 0 || start > a.n_tokens - len || a.pos[start] < 0 ? 0 : len;
}

// Item b of the portions' runs of `toks` tokens (called by a whole warp): info = first token's row, tokens (0: there is no such item), first position, table row
__device__ __forceinline__ void fp8_find_tokens(const Fp8Attn& a, int b, int toks, int* info) {
    int s, item, start = 0, len = 0, pos = 0, slot = 0;
    const bool found = fp8_find(b, a.n_seqs, [&](int i) {
        start = a.seqs[i];
        len = a.seqs[a.seqs_stride + i];
        if (len <= 0 || start < 0 || start > a.n_tokens - len) return 0;
        pos = a.pos[start];
        slot = a.slot[start];
        return pos < 0 ? 0 : (len + toks - 1) / toks;
    }, s, item);
    if (found ? (int)(threadIdx.x & 31) == (s & 31) : (threadIdx.x & 31) == 0) {
        info[0] = start + item * toks;
        info[1] = found ? min(toks, len - item * toks) : 0;
        info[2] = pos + item * toks;
        info[3] = slot;
    }
}

// ------------------------------------------------------------------------------------------------ CUDA cores: any head size up to 256, fp32 or bf16
// A CTA of 8 warps owns up to 32 rows = (token, query head) pairs of one portion and one key/value head, a warp up to four of them, so that a key or value read from shared memory serves
// them all; a decode step's few rows go to as many warps (ROWS 1 or 2 a warp).  Tiles of 32 keys in shared memory as fp32 (code * scale, exact), the next tile's codes on their way in registers meanwhile (VEC: head sizes of whole 16 codes): lane = key for the
// scores, lane = value column for the weighted sum; a running maximum per row, natural exponentials, sums kept by lanes until the end.
// Bound by fp32 products: 2 d FMAs a key and row, 5 shared-memory loads of 16 bytes for 16 of them.
constexpr int kFgTile = 32, kFgWarps = 8, kFgPieces = 4;
struct FgMisc { int info[4], bad[2]; };
__host__ __device__ inline int fg_heads(int R) {      // heads of a group that one CTA's rows take: the largest divisor of the group up to 32
    for (int h = R < 32 ? R : 32; h > 1; h--)
        if (R % h == 0) return h;
    return 1;
}
__host__ __device__ inline int fg_pitch(int d) { return d % 4 ? d | 1 : d + 4; }      // floats of a key's row: neighbouring rows meet in no bank
static size_t fg_smem(int d, int dv, int rows) { return ((size_t)kFgTile * fg_pitch(d) + (size_t)kFgTile * dv + (size_t)rows * kFgWarps * ((d + 3) / 4 * 4 + kFgTile)) * sizeof(float); }

template <typename T, int NC, bool VEC, int ROWS> __global__ void __launch_bounds__(256, 2) fp8_attn_kernel(const Fp8Attn a, int RH) {
    extern __shared__ __align__(16) float fg_smem_raw[];
    __shared__ FgMisc misc;
    const int d = a.d, dv = a.dv, ps = a.pages.page_size, R = a.H / a.G, hblocks = R / RH, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pitch = fg_pitch(d), qp = (d + 3) / 4 * 4;
    const int g = blockIdx.y / hblocks, h0 = g * R + (blockIdx.y % hblocks) * RH;
    griddep_launch_dependents();
    griddep_wait();
    if (warp == 0) fp8_find_tokens(a, blockIdx.x, a.ctoks, misc.info);
    if (threadIdx.x < 2) misc.bad[threadIdx.x] = 0;
    __syncthreads();
    const int tok0 = misc.info[0], ntok = misc.info[1], pos0 = misc.info[2], slot = misc.info[3], max_pos = pos0 + ntok - 1;
    if (ntok <= 0) return;
    const int lo = fp8_first_visible(pos0, a.window, a.chunk), lo_al = lo & ~(a.align - 1);
    const bool cut = a.part > 0 && max_pos + 1 - lo_al > a.part;
    const int k_lo = max(lo, lo_al + (int)blockIdx.z * a.part), k_hi = cut ? min(max_pos + 1, lo_al + (int)(blockIdx.z + 1) * a.part) : max_pos + 1;
    if (blockIdx.z && (!cut || k_lo >= k_hi)) return;
    float* Ks = fg_smem_raw;
    float* Vs = Ks + kFgTile * pitch;
    float* qs = Vs + kFgTile * dv + warp * ROWS * qp;      // the warp's four rows of queries, then their weights
    float* pw = Vs + kFgTile * dv + kFgWarps * ROWS * qp + warp * ROWS * kFgTile;
    // the warp's rows
    const int rows = ntok * RH;
    int row_pos[ROWS], row_first[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const int i = warp * ROWS + r, tok = i / RH, h = h0 + i % RH;
        const bool live = i < rows;
        row_pos[r] = live ? pos0 + tok : -1;
        row_first[r] = live ? fp8_first_visible(pos0 + tok, a.window, a.chunk) : 0;
        const float sc = live ? (a.head_scale ? a.scale * a.head_scale[h] : a.scale) : 0.f;
        for (int c = lane; c < qp; c += 32) qs[r * qp + c] = live && c < d ? to_f(((const T*)a.q)[((long)(tok0 + tok) * a.H + h) * d + c]) * sc : 0.f;
    }
    __syncwarp();
    // a tile's pieces of 16 codes: first the keys' (d / 16 a key), then the values'
    const int kp = d / 16, vp = dv / 16, pieces = kFgTile * (kp + vp);
    uint4 codes[kFgPieces];
    float scale[kFgPieces];
    auto fetch = [&](int j0) {
#pragma unroll
        for (int i = 0; i < kFgPieces; i++) {
            const int at = threadIdx.x + 256 * i;
            scale[i] = 0.f;
            codes[i] = make_uint4(0, 0, 0, 0);
            if (at >= pieces) continue;
            const bool is_v = at >= kFgTile * kp;
            const int per = is_v ? vp : kp, u = is_v ? at - kFgTile * kp : at, key = j0 + u / per, piece = u % per;
            const int page = key < k_hi ? a.pages.page(slot, key / ps) : -1;
            if (page < 0) continue;
            const long block = (long)page * a.G + g;
            scale[i] = a.scales[2 * block + is_v];
            codes[i] = *reinterpret_cast<const uint4*>((is_v ? a.v_codes + (block * ps + key % ps) * dv : a.k_codes + (block * ps + key % ps) * d) + 16 * piece);
        }
    };
    auto spread = [&](int buf) {      // to shared memory, and whether a value is NaN
#pragma unroll
        for (int i = 0; i < kFgPieces; i++) {
            const int at = threadIdx.x + 256 * i;
            if (at >= pieces) continue;
            const bool is_v = at >= kFgTile * kp;
            const int per = is_v ? vp : kp, u = is_v ? at - kFgTile * kp : at, key = u / per, piece = u % per;
            float* to = (is_v ? Vs + key * dv : Ks + key * pitch) + 16 * piece;
            const uint32_t w[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
            uint32_t odd = 0;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                odd |= (w[q] & 0x7f7f7f7fu) + 0x01010101u;
                const float2 x = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w[q], __NV_E4M3)));
                const float2 y = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[q] >> 16), __NV_E4M3)));
                *reinterpret_cast<float4*>(to + 4 * q) = make_float4(x.x * scale[i], x.y * scale[i], y.x * scale[i], y.y * scale[i]);
            }
            if (is_v && (odd & 0x80808080u)) misc.bad[buf] = 1;
        }
    };
    auto bring = [&](int j0, int buf) {      // head sizes of any number of codes
        for (int at = threadIdx.x; at < kFgTile * (d + dv); at += 256) {
            const bool is_v = at >= kFgTile * d;
            const int per = is_v ? dv : d, u = is_v ? at - kFgTile * d : at, k = u / per, c = u % per, key = j0 + k;
            const int page = key < k_hi ? a.pages.page(slot, key / ps) : -1;
            float v = 0.f;
            if (page >= 0) {
                const long block = (long)page * a.G + g;
                v = __half2float(__half(__nv_cvt_fp8_to_halfraw((is_v ? a.v_codes : a.k_codes)[(block * ps + key % ps) * per + c], __NV_E4M3))) * a.scales[2 * block + is_v];
            }
            (is_v ? Vs + k * dv : Ks + k * pitch)[c] = v;
            if (is_v && v != v) misc.bad[buf] = 1;
        }
    };
    float acc[ROWS][NC], m[ROWS], l[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++) acc[r][c] = 0.f;
    }
    if (VEC && k_lo < k_hi) fetch(k_lo);
    for (int j0 = k_lo, buf = 0; j0 < k_hi; j0 += kFgTile, buf ^= 1) {
        __syncthreads();      // (the tile before this one has been read)
        if (threadIdx.x == 0) misc.bad[buf ^ 1] = 0;
        if (VEC) spread(buf); else bring(j0, buf);
        __syncthreads();
        const bool bad = misc.bad[buf];
        if (VEC && j0 + kFgTile < k_hi) fetch(j0 + kFgTile);
        if (warp * ROWS >= rows) continue;
        const int key = j0 + lane;
        const bool here = key < k_hi && a.pages.page(slot, key / ps) >= 0;
        float s[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; r++) s[r] = 0.f;
        const float* kr = Ks + lane * pitch;
        if (d % 4 == 0) {
#pragma unroll 4
            for (int c = 0; c < d; c += 4) {
                const float4 k = *reinterpret_cast<const float4*>(kr + c);
#pragma unroll
                for (int r = 0; r < ROWS; r++) {
                    const float4 q = *reinterpret_cast<const float4*>(qs + r * qp + c);
                    s[r] = fmaf(q.x, k.x, s[r]);
                    s[r] = fmaf(q.y, k.y, s[r]);
                    s[r] = fmaf(q.z, k.z, s[r]);
                    s[r] = fmaf(q.w, k.w, s[r]);
                }
            }
        } else {
            for (int c = 0; c < d; c++)
#pragma unroll
                for (int r = 0; r < ROWS; r++) s[r] = fmaf(qs[r * qp + c], kr[c], s[r]);
        }
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            if (a.softcap > 0.f) s[r] = a.softcap * tanhf(s[r] / a.softcap);
            if (!(here && key <= row_pos[r] && key >= row_first[r])) s[r] = -INFINITY;
            const float mn = fmaxf(m[r], warp_max(s[r])), u = mn == -INFINITY ? 0.f : mn, corr = expf(m[r] - u), p = expf(s[r] - u);
            m[r] = mn;
            l[r] = fmaf(l[r], corr, p);
            pw[r * kFgTile + lane] = p;
            if (corr != 1.f) {
#pragma unroll
                for (int c = 0; c < NC; c++) acc[r][c] *= corr;
            }
        }
        __syncwarp();
        if (!bad) {
#pragma unroll 2
            for (int j = 0; j < kFgTile; j += 4) {
                float4 w[ROWS];
#pragma unroll
                for (int r = 0; r < ROWS; r++) w[r] = *reinterpret_cast<const float4*>(pw + r * kFgTile + j);
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    if (lane + 32 * c < dv) {
                        const float* v = Vs + j * dv + lane + 32 * c;
                        const float v0 = v[0], v1 = v[dv], v2 = v[2 * dv], v3 = v[3 * dv];
#pragma unroll
                        for (int r = 0; r < ROWS; r++) acc[r][c] = fmaf(w[r].w, v3, fmaf(w[r].z, v2, fmaf(w[r].y, v1, fmaf(w[r].x, v0, acc[r][c]))));
                    }
                }
            }
        } else {      // a value that is NaN belongs to the rows that weigh it
            for (int j = 0; j < kFgTile; j++)
#pragma unroll
                for (int r = 0; r < ROWS; r++) {
                    const float w = pw[r * kFgTile + j];
#pragma unroll
                    for (int c = 0; c < NC; c++)
                        if (w != 0.f && lane + 32 * c < dv) acc[r][c] = fmaf(w, Vs[j * dv + lane + 32 * c], acc[r][c]);
                }
        }
        __syncwarp();
    }
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        const int i = warp * ROWS + r, tok = i / RH, h = h0 + i % RH;
        if (i >= rows) break;
        float sum = warp_sum(l[r]);
        const long t = tok0 + tok;
        if (cut) {
            float* o = a.partial + ((t * a.H + h) * a.parts + blockIdx.z) * (dv + 2);
            if (lane == 0) { o[0] = m[r]; o[1] = sum; }
#pragma unroll
            for (int c = 0; c < NC; c++)
                if (lane + 32 * c < dv) o[2 + lane + 32 * c] = acc[r][c];
            continue;
        }
        float corr = 1.f;
        if (a.sink) {
            const float mn = fmaxf(m[r], a.sink[h]);
            corr = m[r] == -INFINITY ? 0.f : expf(m[r] - mn);
            sum = sum * corr + (a.sink[h] == mn ? 1.f : expf(a.sink[h] - mn));
        }
        const float inv = sum > 0.f || sum != sum ? corr * a.out_scale / sum : 0.f;
        T* out = (T*)a.out + t * a.out_stride + (long)h * dv;
#pragma unroll
        for (int c = 0; c < NC; c++)
            if (lane + 32 * c < dv) out[lane + 32 * c] = from_f<T>(acc[r][c] * inv);
    }
}

// The parts of a cut key range, one CTA for each (token, head): the parts' weights once in shared memory (a part without a key has maximum -inf and weighs nothing; the sink joins
// the sum), then 128 columns side by side and the parts dealt among kMergeGroups groups of threads, so that the loads of a long range's parts are all under way at once; the groups' sums are
// added in order.  `unit`: what turns a difference of maxima into a power of two.
constexpr int kMergeGroups = 4;
template <typename T> __global__ void __launch_bounds__(128 * kMergeGroups) fp8_merge_kernel(const Fp8Attn a, float unit) {
    __shared__ float wgt[kFp8MaxParts], red[4], sums[kMergeGroups][128];
    __shared__ int count;
    const long row = blockIdx.x;
    const int t = (int)(row / a.H), h = (int)(row % a.H), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, dv = a.dv, column = tid & 127, group = tid >> 7;
    if (tid == 0) count = 0;
    __syncthreads();
    griddep_launch_dependents();
    griddep_wait();
    // the parts of the range that the token's CTA was cut by (none: a token of no portion, or a range in one piece)
    for (int s = tid; s < a.n_seqs; s += blockDim.x) {
        const int len = fp8_portion(a, s), i = t - a.seqs[s];
        if (i >= 0 && i < len) {
            const int i0 = i / a.ctoks * a.ctoks, p0 = a.pos[a.seqs[s]] + i0, first = fp8_first_visible(p0, a.window, a.chunk) & ~(a.align - 1), n = p0 + min(a.ctoks, len - i0) - first;
            if (n > a.part) count = (n + a.part - 1) / a.part;
        }
    }
    __syncthreads();
    const int parts = min(count, a.parts);
    if (parts == 0) return;
    const float* part = a.partial + row * a.parts * (dv + 2);
    if (group == 0) {      // (four warps)
        const float ms = tid < parts ? part[(long)tid * (dv + 2)] : -INFINITY, ls = tid < parts ? part[(long)tid * (dv + 2) + 1] : 0.f;
        const float top = warp_max(ms);
        if (lane == 0) red[warp] = top;
        asm volatile("barrier.cta.sync 1, 128;" ::: "memory");
        const float sink = a.sink ? a.sink[h] * (kLog2e / unit) : -INFINITY, m = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), sink);
        asm volatile("barrier.cta.sync 1, 128;" ::: "memory");
        const float e = ms > -INFINITY ? exp2f((ms - m) * unit) : 0.f, part_l = warp_sum(ms > -INFINITY ? ls * e : ls);      // (scores of NaN have a sum of NaN and no maximum)
        if (lane == 0) red[warp] = part_l;
        asm volatile("barrier.cta.sync 1, 128;" ::: "memory");
        float l = (red[0] + red[1]) + (red[2] + red[3]);
        if (a.sink) l += sink == m ? 1.f : exp2f((sink - m) * unit);      // (an infinite one too)
        if (tid < parts) wgt[tid] = l > 0.f || l != l ? e / l : 0.f;
        if (l != l && tid < parts) wgt[tid] = l;
    }
    __syncthreads();
    T* out = (T*)a.out + t * a.out_stride + (long)h * dv;
    for (int c0 = 0; c0 < dv; c0 += 128) {
        const int c = c0 + column;
        float acc = 0.f;
        if (c < dv) {
#pragma unroll 16
            for (int s = group; s < parts; s += kMergeGroups) acc = fmaf(wgt[s], part[(long)s * (dv + 2) + 2 + c], acc);
        }
        sums[group][column] = acc;
        __syncthreads();
        if (group == 0 && c < dv) {
            acc = (sums[0][column] + sums[1][column]) + (sums[2][column] + sums[3][column]);
            out[c] = from_f<T>(acc * a.out_scale);
        }
        __syncthreads();
    }
}

}  // namespace ktb
#include "fp8_attn_mma.cuh"
#include "fp8_attn_tc.cuh"
#include "fp8_attn_prompt.cuh"

using namespace ktb;

// Which kernel a call takes, the tokens and query heads of its CTAs, how far a range's start is rounded down, and the CTAs that an SM has places for
struct Fp8Form {
    enum { kCuda, kMma, kDecode, kPrompt } kernel;
    FmForm mma;
    int ctoks, heads, align, places, rows;      // (rows of a warp: kCuda)
};
static bool fg_vec(const ktb200_fp8_attn_params* c) {      // whole pieces of 16 codes
    return c->dim % 16 == 0 && c->vdim % 16 == 0 && !((reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->v_codes)) & 15);
}
static Fp8Form fp8_form(const ktb200_fp8_attn_params* c, int n_tokens, int dtype, int allow_tensor_cores) {
    const int R = c->heads / c->kv_heads;
    if (allow_tensor_cores && fd_takes(c, n_tokens, dtype)) {
        const int RH = fd_heads(R, c->dim);
        return {Fp8Form::kDecode, {}, 1, RH, c->dim == 64 ? 128 : 64, RH <= 8 && c->dim == 128 ? 3 : 2, 0};
    }
    if (allow_tensor_cores && fp_takes(c, n_tokens, dtype)) return {Fp8Form::kPrompt, {}, 2 * (128 / fm_heads(R)), fm_heads(R), kFpKeys, 1, 0};
    if (allow_tensor_cores && fm_takes(c, dtype)) {
        const FmForm f = fm_form(c, n_tokens);
        return {Fp8Form::kMma, f, f.toks, f.RH, kFmKeys, 3, 0};
    }
    const int RH = fg_heads(R), rows = n_tokens > c->n_seqs || RH > 16 || !fg_vec(c) ? 4 : RH > 8 ? 2 : 1;
    return {Fp8Form::kCuda, {}, kFgWarps * rows / RH, RH, 16, 2, rows};
}
// the most keys that a CTA's tokens see together, from a multiple of the alignment on
static long fp8_range(const ktb200_fp8_attn_params* c, int max_keys, const Fp8Form& f) {
    long n = max_keys;
    if (c->window > 0) n = std::min<long>(n, (long)c->window + f.ctoks);
    if (c->chunk > 0) n = std::min<long>(n, (long)c->chunk + f.ctoks);
    return n + f.align;
}
static long fp8_tiles(const ktb200_fp8_attn_params* c, int n_tokens, int ctoks) { return std::min<long>(n_tokens, (long)c->n_seqs + n_tokens / ctoks); }
static bool fp8_sizes_ok(const ktb200_fp8_attn_params* c) { return c && c->heads > 0 && c->kv_heads > 0 && c->heads % c->kv_heads == 0; }

// How a call's ranges are cut: `even` CTAs of a cluster for each, or parts of `part` keys, or (0, 0) not at all.  Not where the CTAs of uncut ranges fill the SMs' places four times.  A
// cluster where eight CTAs a range fill the places once, or leave them 1024 keys at most: as many as fill the places twice and still have 256 keys each (64 contexts of 4095 to 8190: two CTAs a range 148 us; when that was 151, three took 154 and four 158).  Else parts of such a length
// that one round of CTAs covers the ranges, between sequences that decode (whose ranges may have any length) no more than 2048
struct Fp8Cut { int even, part; };
static Fp8Cut fp8_cut(const ktb200_fp8_attn_params* c, int n_tokens, int max_keys, const Fp8Form& f) {
    const int R = c->heads / c->kv_heads;
    const long range = fp8_range(c, max_keys, f), places = f.places * 148, ctas = fp8_tiles(c, n_tokens, f.ctoks) * c->kv_heads * ((R + f.heads - 1) / f.heads);
    if (ctas >= 4 * places || range <= 2 * kFp8MinPart) return {0, 0};
    if (f.kernel == Fp8Form::kDecode && (ctas * kFdCluster >= places || range <= 1024 * kFdCluster))
        return {(int)std::min<long>({kFdCluster, (2 * places + ctas - 1) / ctas, (range + kFp8MinPart - 1) / kFp8MinPart}), 0};
    long part = (range * ctas + places - 1) / places;
    if (c->n_seqs > 1 && f.kernel != Fp8Form::kPrompt) part = std::min<long>(part, 2048);
    part = std::max<long>({part, kFp8MinPart, (range + kFp8MaxParts - 1) / kFp8MaxParts});
    part = (part + 127) / 128 * 128;
    return {0, part < range ? (int)part : 0};
}

static size_t fp8_workspace(const ktb200_fp8_attn_params* c, int n_tokens, int max_keys, int part, const Fp8Form& f) {
    const long parts = part > 0 ? (fp8_range(c, max_keys, f) + part - 1) / part : 1;
    return parts > 1 ? (size_t)n_tokens * c->heads * parts * (c->vdim + 2) * sizeof(float) : 0;
}

extern "C" size_t ktb200_fp8_cache_attn_workspace(const ktb200_fp8_attn_params* c, int n_tokens, int max_keys, int part, int dtype, int allow_tensor_cores) {
    if (!fp8_sizes_ok(c) || n_tokens <= 0) return 0;
    const Fp8Form f = fp8_form(c, n_tokens, dtype, allow_tensor_cores);
    return fp8_workspace(c, n_tokens, max_keys, part < 0 ? fp8_cut(c, n_tokens, max_keys, f).part : part, f);
}

extern "C" int ktb200_fp8_cache_attn(const ktb200_fp8_attn_params* c, int n_tokens, int max_keys, int part, float* workspace, size_t workspace_bytes, int dtype, int allow_tensor_cores,
                                     void* stream) {
    if (!fp8_sizes_ok(c) || c->dim <= 0 || c->dim > kFp8MaxDim || c->vdim <= 0 || c->vdim > kFp8MaxDim || c->page_size <= 0 || c->max_pages <= 0 || c->n_pages < 0 || c->n_slots <= 0 ||
        c->n_seqs < 0 || c->window < 0 || c->chunk < 0 || c->out_stride < (long)c->heads * c->vdim) {
        set_error("fp8_cache_attn: bad argument (head sizes up to %d)", kFp8MaxDim);
        return KTB200_EINVAL;
    }
    if (dtype != KTB200_TYPE_BF16 && dtype != KTB200_TYPE_F32) { set_error("fp8_cache_attn: dtype must be bf16 or f32"); return KTB200_EINVAL; }
    if (part < -1 || (part > 0 && part % 128) || max_keys < 0) { set_error("fp8_cache_attn: part %d (a multiple of 128, 0 or -1), max_keys %d", part, max_keys); return KTB200_EINVAL; }
    if (n_tokens <= 0 || c->n_seqs == 0) return KTB200_OK;
    if (!c->q || !c->pos || !c->slot || !c->seqs || !c->page_table || !c->k_codes || !c->v_codes || !c->scales || !c->out) { set_error("fp8_cache_attn: null pointer"); return KTB200_EINVAL; }
    const bool bf16 = dtype == KTB200_TYPE_BF16;
    const int R = c->heads / c->kv_heads;
    const Fp8Form f = fp8_form(c, n_tokens, dtype, allow_tensor_cores);
    const Fp8Cut own = part < 0 ? fp8_cut(c, n_tokens, max_keys, f) : Fp8Cut{0, part};
    part = own.part;
    const long parts = part ? (fp8_range(c, max_keys, f) + part - 1) / part : 1;
    if (parts > kFp8MaxParts) { set_error("fp8_cache_attn: %ld parts, at most %d", parts, kFp8MaxParts); return KTB200_EINVAL; }
    const size_t need = fp8_workspace(c, n_tokens, max_keys, part, f);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 7))) { set_error("fp8_cache_attn: workspace missing, too small or not aligned"); return KTB200_EINVAL; }
    if ((long)c->kv_heads * R > 65535 || (long)n_tokens * c->heads > 0x7fffffffL) { set_error("fp8_cache_attn: too many heads or tokens"); return KTB200_EINVAL; }
    const cudaStream_t s = (cudaStream_t)stream;
    const Fp8Attn a{c->q, c->heads, c->kv_heads, c->dim, c->vdim, c->scale, c->head_scale, c->softcap, c->window, c->chunk, c->sink, c->out_scale, c->pos, c->slot, c->seqs, c->seqs_stride,
                    c->n_seqs, n_tokens, {c->page_table, c->n_slots, c->max_pages, c->page_size, c->n_pages}, (const uint8_t*)c->k_codes, (const uint8_t*)c->v_codes, c->scales, c->out,
                    c->out_stride, workspace, parts > 1 ? part : 0, (int)parts, own.even > 1 ? own.even : 0, f.ctoks, f.align};
    const dim3 grid((unsigned)fp8_tiles(c, n_tokens, f.ctoks), c->kv_heads * ((R + f.heads - 1) / f.heads), own.even > 1 ? (unsigned)own.even : (unsigned)parts);
    if (f.kernel == Fp8Form::kDecode) {
        const int rc = fd_launch(a, f.heads, grid, s);
        if (rc) return rc;
    } else if (f.kernel == Fp8Form::kPrompt) {
        const int rc = fp_launch(a, f.heads, grid, s);
        if (rc) return rc;
    } else if (f.kernel == Fp8Form::kMma) {
        KTB_CUDA_CHECK(fm_launch(a, f.mma, grid, s));
    } else {
        const size_t smem = fg_smem(c->dim, c->vdim, f.rows);
        const int cols = (c->vdim + 31) / 32;
#define FG_OF(T, NC) (f.rows == 1 ? fp8_attn_kernel<T, NC, true, 1> : f.rows == 2 ? fp8_attn_kernel<T, NC, true, 2> : fg_vec(c) ? fp8_attn_kernel<T, NC, true, 4> : fp8_attn_kernel<T, NC, false, 4>)
        const auto kernel = bf16 ? (cols <= 2 ? FG_OF(__nv_bfloat16, 2) : cols <= 4 ? FG_OF(__nv_bfloat16, 4) : FG_OF(__nv_bfloat16, 8))
                                 : (cols <= 2 ? FG_OF(float, 2) : cols <= 4 ? FG_OF(float, 4) : FG_OF(float, 8));
#undef FG_OF
        KTB_CUDA_CHECK(raise_smem_limit((const void*)kernel, smem));
        KTB_CUDA_CHECK(launch_pdl(kernel, grid, dim3(kFgWarps * 32), smem, s, a, f.heads));
    }
    count_launch();
    if (parts > 1) {
        KTB_CUDA_CHECK(launch_pdl(bf16 ? fp8_merge_kernel<__nv_bfloat16> : fp8_merge_kernel<float>, dim3((unsigned)((long)n_tokens * c->heads)), dim3(128 * kMergeGroups), (size_t)0, s, a,
                                  f.kernel == Fp8Form::kCuda ? kLog2e : 1.0f));
        count_launch();
    }
    return KTB200_OK;
}
