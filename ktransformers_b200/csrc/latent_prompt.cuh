// Expanded attention on tcgen05: a CTA owns up to 256 tokens of one portion and one head as two row tiles of 128; keys run in tiles of 128.
//     s = [q_nope | q_rot] . [k | k_rot] scale,  o = sum p v / sum p          (k, v: latent_expand.cuh's, k_rot: the gathered rows')
//     warp 0          TMA: queries once; keys and values through a FIFO ring of 16 KB blocks: a tile's keys as runs of 64 columns (128 keys x 64), then its values as runs of 64 keys
//     warp 1          MMAs: S = Q K^T from shared memory, O += P V with P in tensor memory.  Of the two row tiles one's products run while the other's soft-max does
//     warps 4-7       soft-max of the first row tile, 8-11 of the second: a thread owns a row.  P (bf16: as values are, each weight 2^-9 of itself off) replaces its S in tensor memory, in two
//                     halves, so that the first half's values are multiplied while the second half's exponentials are made
// The running maximum is only raised, and O scaled in tensor memory, when a tile's outgrows it by 2^8: weights stay below 2^8, sums are fp32.
// TMEM: [S0 | O0 | S1 | O1], 128 columns each.  Shared memory: queries 96 KB, ring 128 KB (nope_dim 64: 64 and 160 KB).
// Where there are few query tiles and heads the keys are cut into parts (blockIdx.z), which latent_merge_kernel joins.
#pragma once
#include "latent_attn.cuh"

namespace ktb {

constexpr int kLpThreads = 384, kLpBlock = 16384, kLpRoom = 229376;      // bytes of a ring block; of queries and ring
constexpr long kLpFits = 96l << 20;
struct LpMaps { CUtensorMap q, q_rot, k, k_rot, v; };
struct LpMisc {
    unsigned long long q_full, full[12], free[12], s_full[2], p_full[2][2], o_done[2];
    uint32_t tmem_base;
};
constexpr int kLpSmem = kLpRoom + 2048 + 1024;
static_assert(sizeof(LpMisc) <= 2048 && kLpSmem <= 232448, "shared memory budget");

struct LatentPrompt {
    const int* plan;
    const uint32_t *bad, *gone;      // a bit a gathered row: who sees it is NaN; nobody sees it
    int n_seqs, heads, pass, part, parts;      // keys of a part (a multiple of 128; 0: one part)
    float scale_log2;
    __nv_bfloat16* out;
    long out_stride;
    float *o_part, *ml_part;      // [token][head][part][V], [token][head][part][2]: the maximum (of scores times log2 e) and the sum
};

template <int N, int V> __global__ void __launch_bounds__(kLpThreads, 1) latent_prompt_kernel(const __grid_constant__ LpMaps maps, const LatentPrompt a) {
    using namespace umma;
    constexpr int QB = N / 64 + 1, NB = QB + 2, SLOTS = (kLpRoom - 2 * QB * kLpBlock) / kLpBlock;      // runs of 64 query columns; blocks of a key tile; of the ring
    static_assert(SLOTS <= 12, "barriers");
    extern __shared__ __align__(16) uint8_t lp_smem_raw[];
    const uint32_t raw = smem_u32(lp_smem_raw), base = (raw + 1023u) & ~1023u, ring = base + 2 * QB * kLpBlock;
    LpMisc& misc = *reinterpret_cast<LpMisc*>(lp_smem_raw + (base - raw) + kLpRoom);
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform(tid >> 5);
    griddep_launch_dependents();
    if (tid == 0) {
        bar_init(smem_u32(&misc.q_full), 1);
        for (int i = 0; i < SLOTS; i++) { bar_init(smem_u32(&misc.full[i]), 1); bar_init(smem_u32(&misc.free[i]), 1); }
        for (int t = 0; t < 2; t++) {
            bar_init(smem_u32(&misc.s_full[t]), 1); bar_init(smem_u32(&misc.o_done[t]), 1);
            for (int h = 0; h < 2; h++) bar_init(smem_u32(&misc.p_full[t][h]), 4);
        }
        bar_fence_init();
    }
    griddep_wait();
    const int rows = a.plan[kPlanRows], nqt = a.plan[kPlanTiles], h0 = a.pass * a.plan[kPlanHeads], nh = min(a.plan[kPlanHeads], a.heads - h0);
    if (nh <= 0 || (long)blockIdx.x >= (long)nh * nqt) return;
    // keys and values that all fit in L2: the tiles that see most keys first, of all heads; else a head's tiles are neighbours, so that those that run together share its keys and values
    // (1000 tokens: 108 us in heads' order, 104 so; 2048 behind 2001: 535, and 564 so)
    const bool by_tile = (long)rows * nh * (N + V) * 2 <= kLpFits;
    const int hl = by_tile ? blockIdx.x % nh : blockIdx.x / nqt, h = h0 + hl;
    const int4 item = reinterpret_cast<const int4*>(a.plan + plan_tiles_at(a.n_seqs))[by_tile ? blockIdx.x / nh : blockIdx.x % nqt];
    const int tok0 = item.x, ntok = item.y, pos0 = item.z, row0 = a.plan[kPlanSeqs + item.w], keys = min(pos0 + ntok, a.plan[kPlanSeqs + a.n_seqs + 1 + item.w]);
    const bool cut = a.part > 0;
    const int k_lo = cut ? blockIdx.z * a.part : 0, k_hi = cut ? min(keys, k_lo + a.part) : keys, n = (k_hi - k_lo + kLatentTile - 1) / kLatentTile, tiles = ntok > 128 ? 2 : 1;
    if (n <= 0) return;
    if (warp == 1) tmem_alloc(smem_u32(&misc.tmem_base), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(misc.tmem_base);

    // registers: 168 a thread at launch; a soft-max thread holds a row of 128 scores (2 x 208 + 88 = 3 x 168)
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 1) {
            // ================================================================ products (converged warp)
            constexpr uint32_t idesc_qk = instr_desc(1, 1, 1, 0, 0, 128, 128), idesc_pv = instr_desc(1, 1, 1, 0, 1, 128, V);      // V [key][column]: B MN-major
            int st = 0, ph = 0;      // the ring's next block and its phase
            auto at = [&](int i) { return st + i < SLOTS ? st + i : st + i - SLOTS; };
            auto need = [&](int i) { bar_wait(smem_u32(&misc.full[at(i)]), st + i < SLOTS ? ph : ph ^ 1); };
            auto pass = [&](int i) { if ((st += i) >= SLOTS) { st -= SLOTS; ph ^= 1; } };
            auto scores = [&](int t) {
                const bool last = t == tiles - 1;
#pragma unroll
                for (int c = 0; c < QB; c++) {
                    if (t == 0) { need(c); tc_fence_after(); }
                    mma_f16_x4(tmem + t * 256, smem_desc(base + (t * QB + c) * kLpBlock, 16, 1024, kLayoutSw128), smem_desc(ring + at(c) * kLpBlock, 16, 1024, kLayoutSw128), idesc_qk, c != 0,
                               c == QB - 1 ? smem_u32(&misc.s_full[t]) : 0, last ? smem_u32(&misc.free[at(c)]) : 0);
                }
            };
            bar_wait(smem_u32(&misc.q_full), 0);
#pragma unroll 1
            for (int t = 0; t < tiles; t++) scores(t);
            pass(QB);
            for (int j = 0; j < n; j++) {
                // (this tile's values are the ring's next two blocks, the next tile's keys those behind them)
#pragma unroll 1
                for (int t = 0; t < tiles; t++) {
#pragma unroll
                    for (int v = 0; v < 2; v++) {
                        if (t == 0) need(v);
                        bar_wait(smem_u32(&misc.p_full[t][v]), j & 1);
                        tc_fence_after();
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            mma_f16_ta(tmem + t * 256 + 128, tmem + t * 256 + 32 * v + 8 * k, smem_desc(ring + at(v) * kLpBlock + k * 2048, 8192, 1024, kLayoutSw128), idesc_pv, (j | v | k) != 0);
                        if (t == tiles - 1) mma_commit(smem_u32(&misc.free[at(v)]));
                    }
                    if (j + 1 == n) {
                        mma_commit(smem_u32(&misc.o_done[t]));
                    } else {
                        const int st0 = st, ph0 = ph;
                        pass(2);
                        scores(t);
                        st = st0; ph = ph0;
                    }
                }
                pass(NB);
            }
        } else if (warp == 0 && lane == 0) {
            // ================================================================ copies
            bar_expect_tx(smem_u32(&misc.q_full), tiles * QB * kLpBlock);
            for (int t = 0; t < tiles; t++) {
                for (int c = 0; c < QB - 1; c++) tma_load_2d(base + (t * QB + c) * kLpBlock, &maps.q, smem_u32(&misc.q_full), h * (N + kLatentRot) + c * 64, tok0 + t * 128);
                tma_load_2d(base + (t * QB + QB - 1) * kLpBlock, &maps.q_rot, smem_u32(&misc.q_full), h * kLatentRot, tok0 + t * 128);
            }
            int st = 0, ph = 1;
            auto block = [&](uint32_t bytes) {      // waits for the ring's next block and announces what comes
                bar_wait(smem_u32(&misc.free[st]), ph);
                bar_expect_tx(smem_u32(&misc.full[st]), bytes);
            };
            auto pass = [&] { if (++st == SLOTS) { st = 0; ph ^= 1; } };
            for (int j = 0; j < n; j++) {
                const int r = row0 + k_lo + j * kLatentTile, hr = hl * rows + r;
                for (int c = 0; c < QB; c++, pass()) {
                    block(kLpBlock);
                    if (c < QB - 1) tma_load_2d(ring + st * kLpBlock, &maps.k, smem_u32(&misc.full[st]), c * 64, hr);
                    else tma_load_2d(ring + st * kLpBlock, &maps.k_rot, smem_u32(&misc.full[st]), kLatent, r);
                }
                for (int v = 0; v < 2; v++, pass()) {
                    block(V * 128);
                    for (int c = 0; c < V / 64; c++) tma_load_2d(ring + st * kLpBlock + c * 8192, &maps.v, smem_u32(&misc.full[st]), N + c * 64, hr + v * 64);
                }
            }
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = (warp - 4) >> 2;
        if (t < tiles) {
            // ================================================================ soft-max
            const int sp = warp & 3, r = 32 * sp + lane, tok = t * 128 + r;
            const uint32_t ts = tmem + ((uint32_t)(32 * sp) << 16) + t * 256, to = ts + 128;
            const int p = pos0 + tok, w_first = pos0 + t * 128 + 32 * sp;      // the row's position and the warp's first
            const bool valid = tok < ntok;
            const float c = a.scale_log2;
            const int odd = a.plan[kPlanOdd];
            float m_ref = -INFINITY, l = 0.f;
            for (int j = 0; j < n; j++) {
                const int k0 = k_lo + j * kLatentTile;
                bar_wait(smem_u32(&misc.s_full[t]), j & 1);
                tc_fence_after();
                float s[128];
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    uint32_t v[32];
                    tmem_ld32(ts + 32 * q, v);
#pragma unroll
                    for (int i = 0; i < 32; i++) s[32 * q + i] = __uint_as_float(v[i]);
                }
                tmem_wait_ld();
                // (the loads above are in registers only now)
#pragma unroll
                for (int i = 0; i < 128; i++) asm volatile("" : "+f"(s[i]));
                if (odd) {
                    const uint4 b = *reinterpret_cast<const uint4*>(a.bad + (row0 + k0) / 32), g = *reinterpret_cast<const uint4*>(a.gone + (row0 + k0) / 32);
                    const uint32_t w[4] = {b.x, b.y, b.z, b.w}, none[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
                    for (int i = 0; i < 128; i++) {
                        if (w[i / 32] >> (i & 31) & 1) s[i] = __int_as_float(0x7fffffff);
                        if (none[i / 32] >> (i & 31) & 1) s[i] = -INFINITY;
                    }
                }
                if (!(k0 + kLatentTile - 1 <= w_first && k0 + kLatentTile <= k_hi)) {
                    const int i1 = min(p, k_hi - 1) - k0;
#pragma unroll
                    for (int i = 0; i < 128; i++)
                        if (i > i1) s[i] = -INFINITY;
                }
                float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int i = 4; i < 128; i += 4)
#pragma unroll
                    for (int q = 0; q < 4; q++) mx[q] = fmaxf(mx[q], s[i + q]);
                const float m_new = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
                const bool raise = m_new > m_ref + 8.f || (m_ref == -INFINITY && m_new > -INFINITY);
                if (__any_sync(0xffffffffu, raise)) {
                    const float alpha = raise ? latent_exp2(m_ref - m_new) : 1.f;
                    if (raise) { m_ref = m_new; l *= alpha; }
                    if (j > 0) {      // (the scores that were waited for are behind the last product into O)
#pragma unroll 1
                        for (int q = 0; q < V / 32; q++) {
                            uint32_t v[32];
                            tmem_ld32(to + 32 * q, v);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
                            tmem_st32(to + 32 * q, v);
                        }
                    }
                }
                const float u = m_ref == -INFINITY ? 0.f : m_ref;
                const f32x2 c2 = pack2(c, c), o2 = pack2(-u, -u);
                f32x2 sum[2] = {0, 0};
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    uint32_t pk[32];
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        float e0, e1;
                        unpack2(fma2(pack2(s[64 * half + 2 * i], s[64 * half + 2 * i + 1]), c2, o2), e0, e1);
                        e0 = latent_exp2(e0);
                        e1 = latent_exp2(e1);
                        pk[i] = latent_pack(e0, e1);
                        sum[i & 1] = add2(sum[i & 1], pack2(e0, e1));
                    }
                    tmem_st32(ts + 32 * half, pk);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(smem_u32(&misc.p_full[t][half]));
                }
                float a0, a1, a2, a3;
                unpack2(sum[0], a0, a1);
                unpack2(sum[1], a2, a3);
                l += (a0 + a1) + (a2 + a3);
            }
            bar_wait(smem_u32(&misc.o_done[t]), 0);
            tc_fence_after();
            const long row = (long)(tok0 + tok) * a.heads + h;
            float k = 1.f;
            l = latent_sum(l, odd & kOddGone);
            if (!cut) k = latent_inverse(l);
            else if (valid) *reinterpret_cast<float2*>(a.ml_part + (row * a.parts + blockIdx.z) * 2) = make_float2(m_ref, l);
            __nv_bfloat16* out = a.out + (long)(tok0 + tok) * a.out_stride + (long)h * V;
            const bool vec = (reinterpret_cast<uintptr_t>(out) & 31) == 0;
#pragma unroll 1
            for (int q = 0; q < V / 32; q++) {
                uint32_t v[32];
                tmem_ld32(to + 32 * q, v);
                tmem_wait_ld();
                if (!valid) continue;
                if (cut) {
                    float4* part = reinterpret_cast<float4*>(a.o_part + (row * a.parts + blockIdx.z) * V + 32 * q);
#pragma unroll
                    for (int i = 0; i < 8; i++) part[i] = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]), __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
                    continue;
                }
                uint32_t o[16];
#pragma unroll
                for (int i = 0; i < 16; i++) o[i] = latent_pack(__uint_as_float(v[2 * i]) * k, __uint_as_float(v[2 * i + 1]) * k);
                if (vec) {
#pragma unroll
                    for (int i = 0; i < 2; i++) latent_store32(out + 32 * q + 16 * i, o + 8 * i);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i++) reinterpret_cast<uint16_t*>(out)[32 * q + i] = (uint16_t)(o[i >> 1] >> (16 * (i & 1)));
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// joins the parts: a warp a token and head, grid (query tiles, heads of the pass, 4), a quarter of the tile's tokens each
template <int V> __global__ void __launch_bounds__(256) latent_merge_kernel(const LatentPrompt a) {
    griddep_launch_dependents();
    griddep_wait();
    const int nqt = a.plan[kPlanTiles], h0 = a.pass * a.plan[kPlanHeads], nh = min(a.plan[kPlanHeads], a.heads - h0), lane = threadIdx.x & 31;
    if ((int)blockIdx.x >= nqt || (int)blockIdx.y >= nh) return;
    const int4 item = reinterpret_cast<const int4*>(a.plan + plan_tiles_at(a.n_seqs))[blockIdx.x];
    const int keys = min(item.z + item.y, a.plan[kPlanSeqs + a.n_seqs + 1 + item.w]), parts = min(a.parts, (keys + a.part - 1) / a.part), h = h0 + blockIdx.y;
    constexpr int C = V / 32;
    for (int i = blockIdx.z * 64 + (threadIdx.x >> 5); i < min(item.y, (int)blockIdx.z * 64 + 64); i += 8) {
        const long row = (long)(item.x + i) * a.heads + h;
        float m = -INFINITY, l = 0.f, o[C];
#pragma unroll
        for (int c = 0; c < C; c++) o[c] = 0.f;
        bool gone = false;
        for (int p = 0; p < parts; p++) m = fmaxf(m, a.ml_part[(row * a.parts + p) * 2]);
#pragma unroll 4
        for (int p = 0; p < parts; p++) {
            const float2 ml = *reinterpret_cast<const float2*>(a.ml_part + (row * a.parts + p) * 2);
            const float w = ml.x == -INFINITY ? 0.f : latent_exp2(ml.x - m);
            const float* src = a.o_part + (row * a.parts + p) * V + lane * C;
            float v[C];
            if (C == 4) {
                const float4 u = *reinterpret_cast<const float4*>(src);
                v[0] = u.x; v[1] = u.y; v[2 % C] = u.z; v[3 % C] = u.w;
            } else {
                const float2 u = *reinterpret_cast<const float2*>(src);
                v[0] = u.x; v[1] = u.y;
            }
            gone |= __float_as_uint(ml.y) == kNoKeys;
            l += ml.x == -INFINITY && ml.y == 0.f ? 0.f : ml.y * w;
#pragma unroll
            for (int c = 0; c < C; c++) o[c] += w == 0.f ? 0.f : v[c] * w;
        }
        const float k = latent_inverse(latent_sum(l, gone));
        __nv_bfloat16* out = a.out + (long)(item.x + i) * a.out_stride + (long)h * V + lane * C;
#pragma unroll
        for (int c = 0; c < C; c++) out[c] = __float2bfloat16_rn(o[c] * k);
    }
}

}  // namespace ktb
