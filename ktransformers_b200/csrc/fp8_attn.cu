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
constexpr int kFp8MaxParts = 128, kFp8MinPart = 256;

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
// grid (tokens, G * head blocks, splits); a warp per query head, the CTA's heads share one key/value head.  Tiles of 32 keys in shared memory as fp32 (code * scale, exact):
// lane = key for the scores, lane = value column for the weighted sum; running maximum and sum per warp, natural exponentials.
constexpr int kFgTile = 32, kFgCols = 8;
template <typename T> __global__ void __launch_bounds__(256) fp8_attn_kernel(const Fp8Attn a) {
    extern __shared__ __align__(16) float fg_smem[];
    __shared__ int info[4];
    const int HB = blockDim.x >> 5, R = a.H / a.G, hblocks = (R + HB - 1) / HB, d = a.d, dv = a.dv, ps = a.pages.page_size;
    const int g = blockIdx.y / hblocks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = (blockIdx.y % hblocks) * HB + warp, h = g * R + r;
    const bool live = r < R;
    griddep_launch_dependents();
    griddep_wait();
    if (warp == 0) fp8_find_tokens(a, blockIdx.x, 1, info);
    __syncthreads();
    if (info[1] <= 0) return;
    const int p = info[2], slot = info[3];
    const long t = info[0];
    float* qs = fg_smem;
    float* Ks = qs + HB * d;
    float* Vs = Ks + kFgTile * (d + 1);
    float* pw = Vs + kFgTile * dv;
    const int lo = fp8_first_visible(p, a.window, a.chunk), lo16 = lo & ~(a.align - 1);
    const bool cut = a.part > 0 && p + 1 - lo16 > a.part;
    const int k_lo = max(lo, lo16 + (int)blockIdx.z * a.part), k_hi = cut ? min(p + 1, lo16 + (int)(blockIdx.z + 1) * a.part) : p + 1;
    if (blockIdx.z && (!cut || k_lo >= k_hi)) return;
    float acc[kFgCols];
#pragma unroll
    for (int c = 0; c < kFgCols; c++) acc[c] = 0.f;
    float m = -INFINITY, l = 0.f;
    if (live) {
        const float sc = a.head_scale ? a.scale * a.head_scale[h] : a.scale;
        for (int i = lane; i < d; i += 32) qs[warp * d + i] = to_f(((const T*)a.q)[(t * a.H + h) * d + i]) * sc;
    }
    for (int j0 = k_lo; j0 < k_hi; j0 += kFgTile) {
        __syncthreads();
        const int nk = min(kFgTile, k_hi - j0);
        unsigned here = 0;      // keys of the tile whose pages are there
        for (int j = 0; j < nk; j++) {
            const int kp = j0 + j, page = a.pages.page(slot, kp / ps);
            if (page < 0) {
                for (int i = threadIdx.x; i < dv; i += blockDim.x) Vs[j * dv + i] = 0.f;
                continue;
            }
            here |= 1u << j;
            const long block = (long)page * a.G + g;
            const float ks = a.scales[2 * block], vs = a.scales[2 * block + 1];
            const uint8_t *k = a.k_codes + (block * ps + kp % ps) * d, *v = a.v_codes + (block * ps + kp % ps) * dv;
            for (int i = threadIdx.x; i < d; i += blockDim.x) Ks[j * (d + 1) + i] = __half2float(__half(__nv_cvt_fp8_to_halfraw(k[i], __NV_E4M3))) * ks;
            for (int i = threadIdx.x; i < dv; i += blockDim.x) Vs[j * dv + i] = __half2float(__half(__nv_cvt_fp8_to_halfraw(v[i], __NV_E4M3))) * vs;
        }
        __syncthreads();
        if (!live) continue;
        float s = -INFINITY;
        if (here >> lane & 1) {
            float q_k = 0.f;
            const float *kr = Ks + lane * (d + 1), *qr = qs + warp * d;
            for (int i = 0; i < d; i++) q_k = fmaf(qr[i], kr[i], q_k);
            s = a.softcap > 0.f ? a.softcap * tanhf(q_k / a.softcap) : q_k;
        }
        const float mn = fmaxf(m, warp_max(s)), u = mn == -INFINITY ? 0.f : mn;
        const float corr = expf(m - u), pj = expf(s - u);
        l = l * corr + warp_sum(pj);
        m = mn;
        pw[warp * kFgTile + lane] = pj;
        __syncwarp();
#pragma unroll
        for (int c = 0; c < kFgCols; c++) acc[c] *= corr;
        for (int j = 0; j < nk; j++) {
            const float wj = pw[warp * kFgTile + j];
#pragma unroll
            for (int c = 0; c < kFgCols; c++)
                if (lane + 32 * c < dv) acc[c] = fmaf(wj, Vs[j * dv + lane + 32 * c], acc[c]);
        }
        __syncwarp();
    }
    if (!live) return;
    if (cut) {
        float* o = a.partial + ((t * a.H + h) * a.parts + blockIdx.z) * (dv + 2);
        if (lane == 0) { o[0] = m; o[1] = l; }
#pragma unroll
        for (int c = 0; c < kFgCols; c++)
            if (lane + 32 * c < dv) o[2 + lane + 32 * c] = acc[c];
        return;
    }
    if (a.sink) {
        const float mn = fmaxf(m, a.sink[h]), corr = expf(m - mn);
        l = l * corr + expf(a.sink[h] - mn);
#pragma unroll
        for (int c = 0; c < kFgCols; c++) acc[c] *= corr;
    }
    const float inv = l > 0.f || l != l ? a.out_scale / l : 0.f;
    T* out = (T*)a.out + t * a.out_stride + (long)h * dv;
#pragma unroll
    for (int c = 0; c < kFgCols; c++)
        if (lane + 32 * c < dv) out[lane + 32 * c] = from_f<T>(acc[c] * inv);
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
        if (a.sink) l += exp2f((sink - m) * unit);
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
    int ctoks, heads, align, places;
};
static Fp8Form fp8_form(const ktb200_fp8_attn_params* c, int n_tokens, int dtype, int allow_tensor_cores) {
    const int R = c->heads / c->kv_heads;
    if (allow_tensor_cores && fd_takes(c, n_tokens, dtype)) return {Fp8Form::kDecode, {}, 1, fm_heads(R), kFdAlign, 3};
    if (allow_tensor_cores && fp_takes(c, n_tokens, dtype)) return {Fp8Form::kPrompt, {}, 2 * (128 / fm_heads(R)), fm_heads(R), kFpKeys, 1};
    if (allow_tensor_cores && fm_takes(c, dtype)) {
        const FmForm f = fm_form(c, n_tokens);
        return {Fp8Form::kMma, f, f.toks, f.RH, kFmKeys, 3};
    }
    return {Fp8Form::kCuda, {}, 1, std::min(R, 8), 16, 3};
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
// cluster where eight CTAs a range fill the places once, or leave them 1024 keys at most: as many as fill the places twice and still have 256 keys each (64 contexts of 4095 to 8190: two CTAs a range 151 us, three 154, four 158).  Else parts of such a length
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
    if (!fp8_sizes_ok(c) || c->dim <= 0 || c->dim > 32 * kFgCols || c->vdim <= 0 || c->vdim > 32 * kFgCols || c->page_size <= 0 || c->max_pages <= 0 || c->n_pages < 0 || c->n_slots <= 0 ||
        c->n_seqs < 0 || c->window < 0 || c->chunk < 0 || c->out_stride < (long)c->heads * c->vdim) {
        set_error("fp8_cache_attn: bad argument (head sizes up to %d)", 32 * kFgCols);
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
        const int HB = f.heads;
        const size_t smem = ((size_t)HB * c->dim + (size_t)kFgTile * (c->dim + 1) + (size_t)kFgTile * c->vdim + (size_t)HB * kFgTile) * sizeof(float);
        KTB_CUDA_CHECK(raise_smem_limit(bf16 ? (const void*)fp8_attn_kernel<__nv_bfloat16> : (const void*)fp8_attn_kernel<float>, smem));
        KTB_CUDA_CHECK(launch_pdl(bf16 ? fp8_attn_kernel<__nv_bfloat16> : fp8_attn_kernel<float>, grid, dim3(HB * 32), smem, s, a));
    }
    count_launch();
    if (parts > 1) {
        KTB_CUDA_CHECK(launch_pdl(bf16 ? fp8_merge_kernel<__nv_bfloat16> : fp8_merge_kernel<float>, dim3((unsigned)((long)n_tokens * c->heads)), dim3(128 * kMergeGroups), (size_t)0, s, a,
                                  f.kernel == Fp8Form::kCuda ? kLog2e : 1.0f));
        count_launch();
    }
    return KTB200_OK;
}
