// Latent attention of any number of new tokens a sequence over the paged latent cache (ktb200_latent_attn), bf16, latents of 512 + 64 rotated columns.
// Two forms of one sum:
//   expanded (portions)   latent_plan_kernel: where each portion's keys and query tiles go; latent_gather_kernel: its cache rows side by side; latent_expand_kernel: keys and values of them
//                         (2 x 512 (N + V) operations a key and head); latent_prompt_kernel: attention with 2 (N + 64 + V) operations a pair and head
//   absorbed (few tokens) latent_few_prep_kernel: blocks of rows and their keys in one line; absorb_kernel: the queries to the latents; latent_few_kernel: attention with 2 (2 x 512 + 64)
//                         operations a pair and head, latent_few_merge_kernel; absorb_kernel: sums of latents to values
// Keys and values of one call take up to kLxBytes; with more the heads go in passes.
#include <algorithm>
#include <type_traits>

#include "latent_expand.cuh"
#include "latent_few.cuh"
#include "latent_prompt.cuh"
#include "mma_tile.cuh"

namespace ktb {

constexpr size_t kLxBytes = (size_t)2 << 30;
// Tokens a sequence on average from which the expanded form takes less, by the call's keys.  128 heads, absorbed / expanded: 64 tokens behind 1000 66 / 67 us, 96 90 / 68; behind 8000 96 228 / 325,
// 128 292 / 328; behind 30000 128 953 / 1339; 8 x 128 behind 4000 1319 / 1609.  16 heads: 128 behind 1000 51 / 58, behind 30000 146 / 209.  (What the expanded form makes of the keys is the same for
// all numbers of tokens, but with few keys its launches and first tiles are most of it.)  One form for a whole call: portions far from the average take the wrong one (2000 tokens beside 63 decoded
// ones behind 4000 keys 2050 us, in two calls 373)
constexpr int kLatentFew = 144, kLatentFewShort = 64, kLatentShort = 2048;

// ------------------------------------------------------------------------------------------------ plan and rows
// one warp: portions in order, 32 side by side
constexpr int kPlanSort = 256;      // query tiles that are sorted
__global__ void __launch_bounds__(32) latent_plan_kernel(const ktb200_latent_attn_params p, int n_tokens, int row_cap, int tile_cap, long rows_of_heads, int* plan) {
    griddep_wait();
    griddep_launch_dependents();      // (as absorb_kernel: behind the wait)
    const int lane = threadIdx.x;
    int* off = plan + kPlanSeqs;
    int4* tiles = reinterpret_cast<int4*>(plan + plan_tiles_at(p.n_seqs));
    __shared__ int4 held[kPlanSort];
    int rows = 0, nt = 0;
    for (int s0 = 0; s0 < p.n_seqs; s0 += 32) {
        const int s = s0 + lane;
        const LatentPortion portion = s < p.n_seqs ? latent_portion(p, n_tokens, s) : LatentPortion{};
        const int first = portion.first, count = portion.count, pos = portion.pos, keys = min(portion.end, row_cap);
        const int r = (keys + kLatentTile - 1) / kLatentTile * kLatentTile, q = (count + kPlanTokens - 1) / kPlanTokens;
        int rs = r, qs = q;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int a = __shfl_up_sync(0xffffffffu, rs, o), b = __shfl_up_sync(0xffffffffu, qs, o);
            if (lane >= o) { rs += a; qs += b; }
        }
        if (s < p.n_seqs) {
            off[s] = rows + rs - r;
            off[p.n_seqs + 1 + s] = keys;
            for (int i = 0; i < q; i++) {      // the last tokens, which see most keys, first
                const int at = nt + qs - q + i, o = (q - 1 - i) * kPlanTokens;
                const int4 tile = make_int4(first + o, min(kPlanTokens, count - o), pos + o, s);
                if (at < tile_cap) tiles[at] = tile;
                if (at < kPlanSort) held[at] = tile;
            }
        }
        rows += __shfl_sync(0xffffffffu, rs, 31);
        nt += __shfl_sync(0xffffffffu, qs, 31);
    }
    // tiles that see most keys first, so that the last CTAs to start have least to do
    nt = min(nt, tile_cap);
    if (nt <= kPlanSort) {
        __syncwarp();
        for (int i = lane; i < nt; i += 32) {
            const int4 tile = held[i];
            const int keys = tile.z + tile.y;
            int before = 0;
            for (int k = 0; k < nt; k++) {
                const int other = held[k].z + held[k].y;
                before += other > keys || (other == keys && k < i);
            }
            tiles[before] = tile;
        }
    }
    if (lane == 0) {
        off[p.n_seqs] = rows;
        plan[kPlanRows] = rows;
        plan[kPlanHeads] = rows > 0 ? (int)min((long)p.heads, rows_of_heads / rows) : p.heads;
        plan[kPlanTiles] = nt;
        plan[kPlanOdd] = 0;
    }
}

// Rows side by side: 32 a CTA and step, a warp four of them.  Rows behind a portion's last key, and rows that are not there, are zeros, and latents that are not finite (latent_copy_row): a bit a row of
// which of these it is
__global__ void __launch_bounds__(256) latent_gather_kernel(const ktb200_latent_attn_params p, int* plan, __nv_bfloat16* lat, uint32_t* bad, uint32_t* gone) {
    griddep_launch_dependents();
    griddep_wait();
    const int rows = plan[kPlanRows], lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int* off = plan + kPlanSeqs;
    __shared__ uint32_t odd[8][2];
    for (int r0 = blockIdx.x * 32; r0 < rows; r0 += gridDim.x * 32) {
        int seq = -1;      // the last portion that begins at or before this row and has one
        for (int s0 = 0; s0 < p.n_seqs; s0 += 32) {
            const unsigned in = __ballot_sync(0xffffffffu, s0 + lane < p.n_seqs && off[s0 + lane] <= r0 && off[s0 + lane + 1] > r0);
            if (in) { seq = s0 + __ffs(in) - 1; break; }
        }
        uint32_t mine = 0, lost = 0;
        if (seq >= 0) {
            const int key0 = r0 - off[seq], keys = off[p.n_seqs + 1 + seq], slot = p.slot[p.seqs[seq]];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int key = key0 + 4 * warp + i;
                int page = -1;
                if (key < keys) page = p.page_table[(long)slot * p.max_pages + key / p.page_size];
                const bool there = (unsigned)page < (unsigned)p.n_pages;
                if (key < keys && !there) lost |= 1u << (4 * warp + i);
                if (latent_copy_row((const __nv_bfloat16*)p.cache + ((long)page * p.page_size + key % p.page_size) * kLatentRow, there, lat + (long)(r0 + 4 * warp + i) * kLatentRow, true)) mine |= 1u << (4 * warp + i);
            }
        }
        if (lane == 0) { odd[warp][0] = mine; odd[warp][1] = lost; }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t all[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++) { all[0] |= odd[i][0]; all[1] |= odd[i][1]; }
            bad[r0 / 32] = all[0];
            gone[r0 / 32] = all[1];
            if (all[0] | all[1]) atomicOr(plan + kPlanOdd, (all[0] ? kOddBad : 0) | (all[1] ? kOddGone : 0));
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ absorbed form
// C[t][h][:] = A[t][h][:] B_h on mma tiles, fp32 sums, one rounding: a CTA has MT tokens of one head and NB columns, and all of its K in shared memory at once: the product is bound by the
// weights' bytes (16.8 MB each with 128 heads), and all of them are on their way at the start.
//   VALUES = false: A = q_nope (K = N), B_h = W_K,h [N][512];  VALUES = true: A = sums of latents (K = 512), B_h = W_V,h^T, W_V,h [V][512]
// All columns of a head in a CTA where there are heads and token tiles for half of the SMs, blocks of 128 (or 32) where there are not.
// The first also writes which tokens there are (`there`: in a portion that is there); the second leaves the rows of others as they are.
template <int MT, int K, bool VALUES, int NB> struct AbsorbShape {
    static constexpr int WARPS = NB > 128 || (VALUES && NB > 32) ? 16 : 8, KP = K + 8, BP = VALUES ? kLatent + 8 : NB + 8, CP = NB + 8;      // padded rows: neighbouring rows meet in no bank
    static constexpr int WM = MT / 16, COLS = NB / 8, WN = WARPS / WM < COLS ? WARPS / WM : COLS, WK = WARPS / (WM * WN), NT = COLS / WN;      // warps along tokens, columns and K; runs of 8 columns a warp
    static constexpr int A_BYTES = MT * KP * 2, B_BYTES = (VALUES ? NB : K) * BP * 2, SMEM = A_BYTES + B_BYTES;
    static_assert(WM * WN * WK == WARPS && NT >= 1 && (NT == 1 || NT % 2 == 0) && K % (16 * WK) == 0 && MT * CP * 2 <= B_BYTES, "shape");
};
template <int MT, int K, bool VALUES, int NB> __global__ void __launch_bounds__(AbsorbShape<MT, K, VALUES, NB>::WARPS * 32) absorb_kernel(const ktb200_latent_attn_params p, const __nv_bfloat16* A, long a_stride, int a_head,
                                                                                                                                         int width, __nv_bfloat16* out, long out_stride, int n_tokens, int* there) {
    using S = AbsorbShape<MT, K, VALUES, NB>;
    constexpr int THREADS = S::WARPS * 32;
    extern __shared__ __align__(16) uint8_t ab_smem[];
    __nv_bfloat16* As = reinterpret_cast<__nv_bfloat16*>(ab_smem);
    __nv_bfloat16* Bs = reinterpret_cast<__nv_bfloat16*>(ab_smem + S::A_BYTES);
    const int h = blockIdx.y, n0 = blockIdx.x * NB, m0 = blockIdx.z * MT, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const __nv_bfloat16* B = (const __nv_bfloat16*)p.w + ((long)h * (p.nope_dim + p.vdim) + (VALUES ? p.nope_dim + n0 : 0)) * kLatent + (VALUES ? 0 : n0);
    griddep_launch_dependents();
    constexpr int BR = VALUES ? NB : K, BC = (VALUES ? kLatent : NB) / 8;
#pragma unroll 8
    for (int i = tid; i < BR * BC; i += THREADS) cp_async16(Bs + (i / BC) * S::BP + (i % BC) * 8, B + (long)(i / BC) * kLatent + (i % BC) * 8, true);      // (the call's first kernel lets the next ones start behind its own wait: what was ahead of the call is complete)
    griddep_wait();
    constexpr int AC = K / 8;
#pragma unroll 4
    for (int i = tid; i < MT * AC; i += THREADS) {
        const int m = i / AC;
        const bool in = m0 + m < n_tokens;
        cp_async16(As + m * S::KP + (i % AC) * 8, A + (long)(in ? m0 + m : 0) * a_stride + (long)h * a_head + (i % AC) * 8, in);
    }
    if (!VALUES && h == 0 && blockIdx.x == 0) {
        for (int m = warp; m < MT; m += S::WARPS) {
            const int t = m0 + m;
            if (t >= n_tokens) break;
            bool in = false;
            for (int s = lane; s < p.n_seqs; s += 32)
                if (t >= p.seqs[s] && t - p.seqs[s] < p.seqs[p.seqs_stride + s]) in |= latent_portion(p, n_tokens, s).count > 0;
            in = __any_sync(0xffffffffu, in);
            if (lane == 0) there[t] = in;
        }
    }
    cp_async_wait_all();
    __syncthreads();
    const int wm = warp % S::WM, wn = warp / S::WM % S::WN, wk = warp / (S::WM * S::WN);
    float acc[S::NT][4];
#pragma unroll
    for (int i = 0; i < S::NT; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) acc[i][c] = 0.f;
    constexpr int KW = K / S::WK;
#pragma unroll 4
    for (int k = wk * KW; k < (wk + 1) * KW; k += 16) {
        uint32_t a[4];
        ldmatrix_x4(a, As + (wm * 16 + (lane & 15)) * S::KP + k + (lane >> 4) * 8);
        if (S::NT == 1) {
            uint32_t b[4];
            ldmatrix_x4(b, Bs + (wn * 8 + (lane & 7)) * S::BP + k + (lane >> 3 & 1) * 8);
            mma_bf16_16816(acc[0], a, b[0], b[1]);
        } else {
#pragma unroll
            for (int i = 0; i < S::NT; i += 2) {      // 16 columns at a time
                uint32_t b[4];
                const int c = (wn * S::NT + i) * 8;
                if (VALUES) ldmatrix_x4(b, Bs + (c + (lane & 7) + (lane >> 4) * 8) * S::BP + k + (lane >> 3 & 1) * 8);
                else ldmatrix_x4_trans(b, Bs + (k + (lane & 15)) * S::BP + c + (lane >> 4) * 8);
                mma_bf16_16816(acc[i], a, b[0], b[1]);
                mma_bf16_16816(acc[(i + 1) % S::NT], a, b[2], b[3]);
            }
        }
    }
    __syncthreads();      // (the operands are done with)
    if (S::WK > 1) {
        float* part = reinterpret_cast<float*>(ab_smem);
        if (wk > 0)
#pragma unroll
            for (int i = 0; i < S::NT * 4; i++) part[((warp - S::WM * S::WN) * S::NT * 4 + i) * 32 + lane] = acc[i / 4][i % 4];
        __syncthreads();
        if (wk == 0)
#pragma unroll
            for (int k = 1; k < S::WK; k++)
#pragma unroll
                for (int i = 0; i < S::NT * 4; i++) acc[i / 4][i % 4] += part[((warp + (k - 1) * S::WM * S::WN) * S::NT * 4 + i) * 32 + lane];
    }
    // results through shared memory, so that whole lines are written
    __nv_bfloat16* Cs = Bs;
    if (wk == 0) {
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int i = 0; i < S::NT; i++)
                *reinterpret_cast<uint32_t*>(Cs + (wm * 16 + (lane >> 2) + 8 * r) * S::CP + (wn * S::NT + i) * 8 + 2 * (lane & 3)) = latent_pack(acc[i][2 * r], acc[i][2 * r + 1]);
    }
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < MT * (NB / 8); i += THREADS) {
        const int m = i / (NB / 8), c = i % (NB / 8) * 8;
        if (m0 + m >= n_tokens || (VALUES && !there[m0 + m])) continue;
        __nv_bfloat16* to = out + (long)(m0 + m) * out_stride + (long)h * width + n0 + c;
        const uint4 v = *reinterpret_cast<const uint4*>(Cs + m * S::CP + c);
        if ((uintptr_t)to % 16 == 0) {
            *reinterpret_cast<uint4*>(to) = v;
        } else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int x = 0; x < 8; x++) reinterpret_cast<uint16_t*>(to)[x] = (uint16_t)(w[x >> 1] >> (16 * (x & 1)));
        }
    }
}
template <int K, int WIDTH, bool VALUES> static int absorb_launch(const ktb200_latent_attn_params* p, const __nv_bfloat16* A, long a_stride, int a_head, __nv_bfloat16* out, long out_stride, int n, int* there, int sms,
                                                                  cudaStream_t s) {
    auto go = [&](auto mt, auto nb) {
        constexpr int MT = decltype(mt)::value, NB = decltype(nb)::value;
        using S = AbsorbShape<MT, K, VALUES, NB>;
        const auto kernel = absorb_kernel<MT, K, VALUES, NB>;
        KTB_CUDA_CHECK(raise_smem_limit((const void*)kernel, S::SMEM));
        KTB_CUDA_CHECK(launch_pdl(kernel, dim3(WIDTH / NB, p->heads, (n + MT - 1) / MT), dim3(S::WARPS * 32), (size_t)S::SMEM, s, *p, A, a_stride, a_head, WIDTH, out, out_stride, n, there));
        count_launch();
        return KTB200_OK;
    };
    using C16 = std::integral_constant<int, 16>;
    using C32 = std::integral_constant<int, 32>;
    using C64 = std::integral_constant<int, 64>;
    using Part = std::integral_constant<int, VALUES ? 32 : 128>;
    using All = std::integral_constant<int, WIDTH>;
    const int mt = n <= 16 ? 16 : n <= 32 ? 32 : 64;
    const bool all = (long)p->heads * ((n + mt - 1) / mt) * 2 >= sms;
    if (mt == 16) return all ? go(C16(), All()) : go(C16(), Part());
    if (mt == 32) return all ? go(C32(), All()) : go(C32(), Part());
    return all ? go(C64(), All()) : go(C64(), Part());
}

// ------------------------------------------------------------------------------------------------ host
static size_t la_up(size_t n) { return (n + 1023) / 1024 * 1024; }
struct LatentLayout {      // of the workspace: byte offsets, and what the sizes follow from
    int form, rows, tiles, passes, parts, part, pairs, blocks, tail_tiles;
    bool gathered;      // absorbed: pages that are not whole 32 rows are laid side by side first
    size_t plan, lat, bad, gone, kv, o_part, ml_part, few, there, tails, tail_bad, tail_gone, tail_holes, q_abs, sums, total;
    long rows_of_heads;      // expanded rows, one a head, that there is room for
};
static int latent_form(const ktb200_latent_attn_params* p, int n_tokens, int max_kv) {
    if (p->form) return p->form;
    return (long)n_tokens >= (long)(max_kv <= kLatentShort ? kLatentFewShort : kLatentFew) * p->n_seqs ? 2 : 1;
}
static int latent_layout(LatentLayout& y, const ktb200_latent_attn_params* p, int n_tokens, int max_kv) {
    y = LatentLayout{};
    y.form = latent_form(p, n_tokens, max_kv);
    int device = 0;
    KTB_CUDA_CHECK(cudaGetDevice(&device));
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += la_up(n); return o; };
    const size_t H = p->heads, bn = p->nope_dim + p->vdim;
    y.gathered = y.form == 1 && p->page_size % 32 != 0;
    const long tiled = ((long)max_kv + kLatentTile - 1) / kLatentTile * kLatentTile, rows = y.form == 2 || y.gathered ? tiled * p->n_seqs : 0;
    if (rows > (1L << 30)) { set_error("latent_attn: %d sequences of up to %d keys", p->n_seqs, max_kv); return KTB200_EINVAL; }
    y.rows = (int)rows;
    if (y.form == 2 || y.gathered) {
        y.tiles = n_tokens / kPlanTokens + p->n_seqs;
        y.plan = take((plan_tiles_at(p->n_seqs) + 4L * y.tiles) * 4);
        y.lat = take((size_t)rows * kLatentRow * 2);
        y.bad = take((size_t)rows / 32 * 4);
        y.gone = take((size_t)rows / 32 * 4);
    }
    if (y.form == 2) {
        const long room = (long)std::max<size_t>((size_t)rows, std::min(H * (size_t)rows, kLxBytes / (bn * 2)));
        y.rows_of_heads = std::min(room, 0x7fffffffL);
        const long per = y.rows_of_heads / rows;
        y.passes = (int)((H + per - 1) / per);
        y.kv = take((size_t)y.rows_of_heads * bn * 2);
        // few query tiles and heads: the keys in parts of 512 and more, as many as fill the SMs
        const long ctas = (long)y.tiles * std::min((long)H, per), sms = num_sms(device);
        y.parts = 1;
        if (2 * ctas <= sms && tiled > 1024) {
            y.part = (int)std::max(512L, (tiled / (sms / ctas) + kLatentTile - 1) / kLatentTile * kLatentTile);
            y.parts = (int)((tiled + y.part - 1) / y.part);
            if (y.parts == 1) y.part = 0;
        }
        if (y.parts > 1) {
            y.o_part = take((size_t)n_tokens * H * y.parts * p->vdim * 4);
            y.ml_part = take((size_t)n_tokens * H * y.parts * 8);
        }
    } else {
        if ((long)n_tokens * p->heads > (1L << 30)) { set_error("latent_attn: %d tokens of %d heads", n_tokens, p->heads); return KTB200_EINVAL; }
        y.pairs = num_sms(device) / 2;
        y.blocks = (int)((long)n_tokens * p->heads / kFewRows + p->n_seqs);
        y.few = take((few_blocks_at(y.pairs) + (long)y.blocks * (sizeof(FewBlock) / 4)) * 4);
        y.there = take((size_t)n_tokens * 4);
        if (!y.gathered) {
            y.tail_tiles = n_tokens / kFewTile + 2 * p->n_seqs;
            y.tails = take((size_t)y.tail_tiles * kFewTile * kLatentRow * 2);
            y.tail_bad = take((size_t)y.tail_tiles * kFewTile / 8);
            y.tail_gone = take((size_t)y.tail_tiles * kFewTile / 8);
            y.tail_holes = take((size_t)y.tail_tiles * 16);
        }
        y.q_abs = take((size_t)n_tokens * H * kLatent * 2);
        y.sums = take((size_t)n_tokens * H * kLatent * 2);
        y.o_part = take((size_t)2 * y.pairs * kFewRows * kLatent * 4);
        y.ml_part = take((size_t)2 * y.pairs * kFewRows * 8);
    }
    y.total = at;
    return KTB200_OK;
}
static int latent_check(const ktb200_latent_attn_params* p, int max_kv) {
    if (!p || p->heads <= 0 || p->page_size <= 0 || p->max_pages <= 0 || p->n_slots <= 0 || p->n_pages <= 0 || p->n_seqs < 0 || max_kv < 0) { set_error("latent_attn: bad sizes"); return KTB200_EINVAL; }
    if ((p->nope_dim != 64 && p->nope_dim != 128) || (p->vdim != 64 && p->vdim != 128)) { set_error("latent_attn: heads of %d + 64 and values of %d: 64 or 128 of each", p->nope_dim, p->vdim); return KTB200_EINVAL; }
    if (p->form < 0 || p->form > 2) { set_error("latent_attn: form %d", p->form); return KTB200_EINVAL; }
    if (!(p->scale > 0.f) || p->scale > 1e30f) { set_error("latent_attn: the scale has to be above zero"); return KTB200_EINVAL; }
    if (p->q_stride < (long)p->heads * (p->nope_dim + kLatentRot) || p->out_stride < (long)p->heads * p->vdim) { set_error("latent_attn: rows overlap"); return KTB200_EINVAL; }
    if (p->q_stride % 8) { set_error("latent_attn: rows of q have to begin at multiples of 16 bytes"); return KTB200_EINVAL; }
    if ((long)p->n_pages * p->page_size > 0x7fffffffL) { set_error("latent_attn: %d pages of %d tokens", p->n_pages, p->page_size); return KTB200_EINVAL; }
    return KTB200_OK;
}
static int latent_map(CUtensorMap* map, const void* ptr, long width, long rows, long stride, int box_rows) {      // boxes of 64 columns x box_rows, 128-byte swizzled; what is outside comes as zeros
    const umma::EncodeTiledFn enc = umma::encode_tiled();
    if (!enc) { set_error("latent_attn: cuTensorMapEncodeTiled is not available from this driver"); return KTB200_ECUDA; }
    const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    const CUresult cr = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS) { set_error("latent_attn: cuTensorMapEncodeTiled failed (%d)", (int)cr); return KTB200_ECUDA; }
    return KTB200_OK;
}
// the plan and the rows of all portions
static int latent_rows(const ktb200_latent_attn_params* p, const LatentLayout& y, int n_tokens, uint8_t* ws, int sms, cudaStream_t s) {
    int* plan = (int*)(ws + y.plan);
    KTB_CUDA_CHECK(launch_pdl(latent_plan_kernel, dim3(1), dim3(32), (size_t)0, s, *p, n_tokens, (int)(y.rows / p->n_seqs), y.tiles, y.rows_of_heads, plan));
    KTB_CUDA_CHECK(launch_pdl(latent_gather_kernel, dim3(std::min(y.rows / 32, 8 * sms)), dim3(256), (size_t)0, s, *p, plan, (__nv_bfloat16*)(ws + y.lat), (uint32_t*)(ws + y.bad), (uint32_t*)(ws + y.gone)));
    count_launch(2);
    return KTB200_OK;
}
template <int N, int V> static int latent_expanded(const ktb200_latent_attn_params* p, const LatentLayout& y, int n_tokens, uint8_t* ws, int sms, cudaStream_t s) {
    constexpr int BN = N + V;
    const int rc = latent_rows(p, y, n_tokens, ws, sms, s);
    if (rc) return rc;
    CUtensorMap lat, w;
    LpMaps m;
    const __nv_bfloat16 *rows = (const __nv_bfloat16*)(ws + y.lat), *kv = (const __nv_bfloat16*)(ws + y.kv);
    int e = latent_map(&lat, rows, kLatentRow, y.rows, kLatentRow, 128);
    if (!e) e = latent_map(&w, p->w, kLatent, (long)p->heads * BN, kLatent, BN / 2);
    if (!e) e = latent_map(&m.q, p->q, (long)p->heads * (N + kLatentRot), n_tokens, p->q_stride, 128);
    if (!e) e = latent_map(&m.q_rot, p->q_rot, (long)p->heads * kLatentRot, n_tokens, (long)p->heads * kLatentRot, 128);
    if (!e) e = latent_map(&m.k, kv, BN, y.rows_of_heads, BN, 128);
    if (!e) e = latent_map(&m.v, kv, BN, y.rows_of_heads, BN, 64);
    if (e) return e;
    m.k_rot = lat;
    KTB_CUDA_CHECK(raise_smem_limit((const void*)latent_expand_kernel, kLxSmem));
    KTB_CUDA_CHECK(raise_smem_limit((const void*)latent_prompt_kernel<N, V>, kLpSmem));
    const int pairs = sms / 2, mt = (y.rows + 255) / 256;
    const int ctas = (int)std::min<long>((long)y.tiles * p->heads, 0x7fffffffL);
    LatentPrompt a{(const int*)(ws + y.plan), (const uint32_t*)(ws + y.bad), (const uint32_t*)(ws + y.gone), p->n_seqs, p->heads, 0, y.parts > 1 ? y.part : 0, y.parts, p->scale * 1.4426950408889634f, (__nv_bfloat16*)p->out, p->out_stride,
                   (float*)(ws + y.o_part), (float*)(ws + y.ml_part)};
    for (a.pass = 0; a.pass < y.passes; a.pass++) {
        KTB_CUDA_CHECK(launch_pdl(latent_expand_kernel, dim3((unsigned)(2 * std::min<long>((long)mt * p->heads, pairs))), dim3(kLxThreads), (size_t)kLxSmem, s, lat, w, m.k, a.plan, BN,
                                  p->heads, a.pass));
        KTB_CUDA_CHECK(launch_pdl(latent_prompt_kernel<N, V>, dim3(ctas, 1, y.parts), dim3(kLpThreads), (size_t)kLpSmem, s, m, a));
        count_launch(2);
        if (y.parts > 1) {
            KTB_CUDA_CHECK(launch_pdl(latent_merge_kernel<V>, dim3(y.tiles, p->heads, 4), dim3(256), (size_t)0, s, a));
            count_launch();
        }
    }
    return KTB200_OK;
}
template <int N, int V> static int latent_absorbed(const ktb200_latent_attn_params* p, const LatentLayout& y, int n_tokens, uint8_t* ws, int sms, cudaStream_t s) {
    if (y.gathered) {
        const int rc = latent_rows(p, y, n_tokens, ws, sms, s);
        if (rc) return rc;
    }
    __nv_bfloat16 *q_abs = (__nv_bfloat16*)(ws + y.q_abs), *tails = (__nv_bfloat16*)(ws + y.tails);
    int* there = (int*)(ws + y.there);
    const long rows = (long)n_tokens * p->heads, wide = (long)p->heads * kLatent;
    LatentFew a{*p, (int*)(ws + y.few), n_tokens, y.blocks, y.gathered ? 0x7fffffff : y.tail_tiles, y.pairs, p->page_size % 64 && !y.gathered ? 32 : 64, y.gathered ? (const int*)(ws + y.plan) : nullptr,
                (const uint32_t*)(ws + (y.gathered ? y.bad : y.tail_bad)), (const uint32_t*)(ws + (y.gathered ? y.gone : y.tail_gone)), (const uint4*)(ws + y.tail_holes), p->scale * 1.4426950408889634f, (__nv_bfloat16*)(ws + y.sums), (float*)(ws + y.o_part), (float*)(ws + y.ml_part)};
    FewMaps m;
    int e = latent_map(&m.q, q_abs, kLatent, rows, kLatent, 64);
    if (!e) e = latent_map(&m.q_rot, p->q_rot, kLatentRot, rows, kLatentRot, 64);
    if (!e) e = y.gathered ? latent_map(&m.rows, ws + y.lat, kLatentRow, y.rows, kLatentRow, a.box) : latent_map(&m.rows, p->cache, kLatentRow, (long)p->n_pages * p->page_size, kLatentRow, a.box);
    if (!e) e = y.gathered ? latent_map(&m.tails, ws + y.lat, kLatentRow, y.rows, kLatentRow, a.box) : latent_map(&m.tails, tails, kLatentRow, (long)y.tail_tiles * kFewTile, kLatentRow, a.box);
    if (e) return e;
    KTB_CUDA_CHECK(launch_pdl(latent_few_prep_kernel, dim3(1 + (y.gathered ? 0 : 4 * y.tail_tiles)), dim3(256), (size_t)0, s, a, tails, (uint32_t*)(ws + y.tail_bad), (uint32_t*)(ws + y.tail_gone), (uint32_t*)(ws + y.tail_holes)));
    count_launch();
    const int rc = absorb_launch<N, kLatent, false>(p, (const __nv_bfloat16*)p->q, p->q_stride, N + kLatentRot, q_abs, wide, n_tokens, there, sms, s);
    if (rc) return rc;
    KTB_CUDA_CHECK(raise_smem_limit((const void*)latent_few_kernel, kFewSmem));
    KTB_CUDA_CHECK(launch_pdl(latent_few_kernel, dim3(2 * y.pairs), dim3(kFewThreads), (size_t)kFewSmem, s, m, a));
    KTB_CUDA_CHECK(launch_pdl(latent_few_merge_kernel, dim3(y.blocks, kFewRows / 8), dim3(256), (size_t)0, s, a));
    count_launch(2);
    return absorb_launch<kLatent, V, true>(p, a.sums, wide, kLatent, (__nv_bfloat16*)p->out, p->out_stride, n_tokens, there, sms, s);
}

}  // namespace ktb

using namespace ktb;

extern "C" {

int ktb200_latent_attn_form(const ktb200_latent_attn_params* p, int n_tokens, int max_kv) { return p ? latent_form(p, n_tokens, max_kv) : 0; }

size_t ktb200_latent_attn_workspace(const ktb200_latent_attn_params* p, int n_tokens, int max_kv) {
    LatentLayout y;
    if (latent_check(p, max_kv) || n_tokens <= 0 || p->n_seqs == 0 || max_kv == 0 || latent_layout(y, p, n_tokens, max_kv)) return 0;
    return y.total;
}

int ktb200_latent_attn(const ktb200_latent_attn_params* p, int n_tokens, int max_kv, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = latent_check(p, max_kv);
    if (rc) return rc;
    if (n_tokens <= 0 || p->n_seqs == 0) return KTB200_OK;
    if (max_kv == 0) { set_error("latent_attn: %d tokens and no keys", n_tokens); return KTB200_EINVAL; }
    if (!p->q || !p->q_rot || !p->w || !p->pos || !p->slot || !p->seqs || !p->page_table || !p->cache || !p->out) { set_error("latent_attn: null pointer"); return KTB200_EINVAL; }
    if (((uintptr_t)p->q | (uintptr_t)p->q_rot | (uintptr_t)p->w | (uintptr_t)p->cache) & 15) { set_error("latent_attn: q, q_rot, w and the cache have to be 16-byte aligned"); return KTB200_EINVAL; }
    LatentLayout y;
    if ((rc = latent_layout(y, p, n_tokens, max_kv))) return rc;
    if (!workspace || ((uintptr_t)workspace & 1023) || workspace_bytes < y.total) { set_error("latent_attn: workspace of %zu bytes, 1024-byte aligned; %zu are needed", workspace_bytes, y.total); return KTB200_EINVAL; }
    int device = 0;
    KTB_CUDA_CHECK(cudaGetDevice(&device));
    const int sms = num_sms(device);
    uint8_t* ws = (uint8_t*)workspace;
    const cudaStream_t s = (cudaStream_t)stream;
    auto call = [&](auto n, auto v) {
        constexpr int N = decltype(n)::value, V = decltype(v)::value;
        return y.form == 2 ? latent_expanded<N, V>(p, y, n_tokens, ws, sms, s) : latent_absorbed<N, V>(p, y, n_tokens, ws, sms, s);
    };
    using C64 = std::integral_constant<int, 64>;
    using C128 = std::integral_constant<int, 128>;
    if (p->nope_dim == 128) return p->vdim == 128 ? call(C128(), C128()) : call(C128(), C64());
    return p->vdim == 128 ? call(C64(), C128()) : call(C64(), C64());
}

}  // extern "C"
