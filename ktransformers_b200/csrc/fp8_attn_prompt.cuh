// Attention of prompt portions over the paged e4m3 cache on tcgen05 (bf16 queries, heads of 128, pages of whole 64 tokens).
//
// A CTA owns 256 rows = (token, query head) pairs of one sequence portion and one key/value head as two tiles of 128 (RH heads of 128 / RH consecutive tokens each); keys run in
// tiles of 128 from a multiple of 128 on.
//     warps 0, 2, 3   values: TMA brings a tile's codes, the warps turn them into swizzled fp16 operands, which hold every e4m3 number exactly (a conversion for two codes).  Keys need none:
//                     warp 0 has their codes brought as operands
//     warp 1          MMAs of 64 keys at a time: S = Q K^T (kind::f8f6f4) from shared memory, O += P V (kind::f16) with P in tensor memory.  A row tile has two buffers of 64 scores: S of the
//                     next 64 keys is there before the soft-max of these is done, which so never waits for a product
//     warps 4-7       soft-max of the first tile, 8-11 of the second: a thread owns a row.  First it makes its row of Q: moved by a power of two so that its largest stands in [128, 256) and
//                     split into two e4m3 numbers, q = q1 + q2, whose products add up in one sum: exact for bf16 numbers down to 2^-9 of the largest, 2^-17 of it off below.
//                     t = s log2(e) + log2(value scale), p = 2^(t - m), l += p / (value scale): scales are one number a page and head, so that of 64 scores at a time they change the
//                     factor and the offset of an fma that is there anyway, and O needs none.  P (fp16) replaces its S in tensor memory; m is 7 below a row's largest t and raised, and
//                     O scaled in tensor memory, only when a t outgrows it by 15: weights are 2^-11 of themselves off down to 2^-21 of the largest, and 2^-32 of that below
// TMEM: [S0 | O0 | S1 | O1], 128 columns each (S: two buffers of 64).  Shared memory: Q 64 KB, K 3 x 16 KB, V 2 x 32 KB as fp16 and 2 x 16 KB as codes.
// (With keys turned into fp16 as well the three warps were the bound: 2048 tokens behind 2001 took 318 us, 228 with their work left out.)
#pragma once
#include <cuda.h>

#include "umma.cuh"

namespace ktb {

constexpr int kFpThreads = 384, kFpKeys = 128, kFpTile = 128 * 128 * 2, kFpCodes = 128 * 128, kFpKStages = 3, kFpBad = 64;
struct FpMisc {
    unsigned long long q_full, v8_full[2], k_full[kFpKStages], k_free[kFpKStages], v_full[2], v_free[2], s_full[2][2], p_full[2][2], pv_done[2][2];      // [row tile][buffer]
    float2 scales[4][2];      // of a tile's two runs of 64 keys (zeros: not there)
    uint32_t tmem_base;
    int info[4], n_bad, bad_lo, bad_hi;
    int2 bad[kFpBad];      // values that are NaN in tiles that not every row sees whole: (key, run of 16 columns << 16 | which of them)
};
constexpr int kFpSmem = 4 * kFpTile + (kFpKStages + 2) * kFpCodes + (int)sizeof(FpMisc) + 1024;
static_assert(kFpSmem <= 232448, "shared memory budget");

__global__ void __launch_bounds__(kFpThreads, 1) fp8_attn_prompt_kernel(const __grid_constant__ FdMaps maps, const Fp8Attn a, int RH) {
    using namespace umma;
    extern __shared__ __align__(16) uint8_t fp_smem_raw[];
    const uint32_t raw = smem_u32(fp_smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* smem = fp_smem_raw + (base - raw);
    const uint32_t vbase = base + 2 * kFpTile, kbase = base + 4 * kFpTile, v8base = kbase + kFpKStages * kFpCodes;
    FpMisc& misc = *reinterpret_cast<FpMisc*>(smem + 4 * kFpTile + (kFpKStages + 2) * kFpCodes);
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform(tid >> 5), ps = a.pages.page_size, TOKS = 128 / RH, R = a.H / a.G, hblocks = R / RH;
    griddep_launch_dependents();
    if (tid == 0) {
        bar_init(smem_u32(&misc.q_full), 9);
        for (int i = 0; i < kFpKStages; i++) { bar_init(smem_u32(&misc.k_full[i]), 1); bar_init(smem_u32(&misc.k_free[i]), 1); }
        for (int i = 0; i < 2; i++) {
            bar_init(smem_u32(&misc.v8_full[i]), 1); bar_init(smem_u32(&misc.v_full[i]), 3); bar_init(smem_u32(&misc.v_free[i]), 1);
            for (int b = 0; b < 2; b++) { bar_init(smem_u32(&misc.s_full[i][b]), 1); bar_init(smem_u32(&misc.p_full[i][b]), 4); bar_init(smem_u32(&misc.pv_done[i][b]), 1); }
        }
        bar_fence_init();
        misc.n_bad = 0;
        misc.bad_lo = 0x7fffffff;
        misc.bad_hi = -1;
        tma_prefetch_desc(&maps.k);
        tma_prefetch_desc(&maps.v);
    }
    griddep_wait();
    if (warp == 1) fp8_find_tokens(a, gridDim.y - 1 - blockIdx.y, 2 * TOKS, misc.info);      // the last tokens, which see most keys, first
    __syncthreads();
    const int tok0 = misc.info[0], ntok = misc.info[1], pos0 = misc.info[2], slot = misc.info[3];
    if (ntok <= 0) return;
    const int g = blockIdx.x / hblocks, h0 = g * R + (blockIdx.x % hblocks) * RH;
    const int max_pos = pos0 + ntok - 1, lo = fp8_first_visible(pos0, a.window, a.chunk), lo_al = lo & ~(kFpKeys - 1);
    const bool cut = a.part > 0 && max_pos + 1 - lo_al > a.part;
    const int k_lo = lo_al + blockIdx.z * a.part, k_hi = cut ? min(max_pos + 1, k_lo + a.part) : max_pos + 1;
    if (k_lo >= k_hi) return;
    const int n = (k_hi - k_lo + kFpKeys - 1) / kFpKeys;
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
            constexpr uint32_t idesc_qk = instr_desc(1, 0, 0, 0, 0, 128, 64), idesc_pv = instr_desc(1, 0, 0, 0, 1, 128, 128);      // V [key][column]: B MN-major
            int kst = 0, kph = 0;      // the stage and phase of the keys that S takes next
            auto scores = [&](int t, int i) {      // of the i-th 64 keys
                const uint32_t qb = base + t * kFpTile;
                const uint64_t k = smem_desc(kbase + kst * kFpCodes + (i & 1) * (kFpCodes / 2), 16, 1024, kLayoutSw128);
                const uint32_t d = tmem + t * 256 + (i & 1) * 64;
                mma_f8_x4(d, smem_desc(qb, 16, 1024, kLayoutSw128), k, idesc_qk, 0);
                mma_f8_x4(d, smem_desc(qb + kFpCodes, 16, 1024, kLayoutSw128), k, idesc_qk, 1, smem_u32(&misc.s_full[t][i & 1]), t && (i & 1) ? smem_u32(&misc.k_free[kst]) : 0);
            };
            bar_wait(smem_u32(&misc.q_full), 0);
            bar_wait(smem_u32(&misc.k_full[0]), 0);
            tc_fence_after();
#pragma unroll 1
            for (int i = 0; i < 4; i++) scores(i & 1, i >> 1);
            for (int i = 0; i < 2 * n; i++) {
                const int j = i >> 1, st = j & 1, buf = i & 1;
                const uint32_t vb = vbase + st * kFpTile + buf * 4 * 2048;
                if (buf == 0) {
                    bar_wait(smem_u32(&misc.v_full[st]), (j >> 1) & 1);
                    if (++kst == kFpKStages) { kst = 0; kph ^= 1; }
                    if (j + 1 < n) bar_wait(smem_u32(&misc.k_full[kst]), kph);
                }
#pragma unroll 1
                for (int t = 0; t < 2; t++) {
                    bar_wait(smem_u32(&misc.p_full[t][buf]), j & 1);
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        mma_f16_ta(tmem + t * 256 + 128, tmem + t * 256 + buf * 64 + 8 * k, smem_desc(vb + k * 2048, kFpTile / 2, 1024, kLayoutSw128), idesc_pv, (i | k) != 0);
                    mma_commit(smem_u32(&misc.pv_done[t][buf]));
                    if (t == 1 && buf == 1) mma_commit(smem_u32(&misc.v_free[st]));
                    if (j + 1 < n) scores(t, i);      // (of 128 keys on)
                }
            }
        } else {
            // ================================================================ copies, and values' codes to fp16
            const int cw = warp == 0 ? 0 : warp - 1, none = a.pages.n_pages * a.G * ps;      // (rows from `none` on are outside the maps: zeros)
            const bool slot_ok = (unsigned)slot < (unsigned)a.pages.slots;
            const int* pt = a.pages.table + (slot_ok ? (long)slot * a.pages.max_pages : 0);
            const int last_first = fp8_first_visible(max_pos, a.window, a.chunk);
            auto row_of = [&](int key) {      // of a run of 64 keys; `none`: not there, or nobody sees it
                if (!slot_ok || key >= k_hi || key + 64 <= lo) return none;
                const int page = pt[(key / ps) % a.pages.max_pages];
                return (unsigned)page < (unsigned)a.pages.n_pages ? (page * a.G + g) * ps + key % ps : none;
            };
            auto bring = [&](uint32_t dst, const CUtensorMap* map, unsigned long long* bar, int r0, int r1) {
                bar_expect_tx(smem_u32(bar), kFpCodes);
                tma_load_2d(dst, map, smem_u32(bar), 0, r0);
                tma_load_2d(dst + kFpCodes / 2, map, smem_u32(bar), 0, r1);
            };
            // 8 rows and 4 of their 8 pieces of 16 codes at a time, into the operand: two blocks of 64 columns, rows of 128 bytes.  Both sides are 128-byte-swizzled, so that no two of the lanes
            // that read or write together meet in a bank
            auto turn = [&](uint32_t src, uint32_t dst, int k0) {
                const bool partial = !(k0 >= last_first && k0 + kFpKeys - 1 <= pos0), edge = k0 < lo || k0 + kFpKeys > k_hi;
#pragma unroll 4
                for (int i = cw; i < 32; i += 3) {
                    const int r = 8 * (i >> 1) + (lane & 7), piece = 4 * (i & 1) + (lane >> 3);
                    const uint4 v = lds16(src + r * 128 + ((piece ^ (lane & 7)) << 4));
                    uint32_t w[4] = {v.x, v.y, v.z, v.w};
                    if (edge && (k0 + r < lo || k0 + r >= k_hi)) w[0] = w[1] = w[2] = w[3] = 0;      // values that no row sees may be anything (0 x NaN)
                    if (partial) {      // a value that is NaN belongs to the rows that see it: they are told at the end
                        uint32_t mask = 0;
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const uint32_t odd = (((w[q] & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u;
                            mask |= ((odd * 0x10204080u) >> 28) << (4 * q);      // byte b's bit to bit b
                            w[q] &= ~(odd * 0xffu);
                        }
                        if (mask) {
                            const int at = atomicAdd(&misc.n_bad, 1);
                            if (at < kFpBad) misc.bad[at] = make_int2(k0 + r, piece << 16 | (int)mask);
                            atomicMin(&misc.bad_lo, k0 + r);
                            atomicMax(&misc.bad_hi, k0 + r);
                        }
                    }
                    uint32_t f[8];
#pragma unroll
                    for (int q = 0; q < 4; q++) { f[2 * q] = f16_of_codes(w[q]); f[2 * q + 1] = f16_of_codes(w[q] >> 16); }
                    const uint32_t at = dst + (i & 1) * (kFpTile / 2) + r * 128;
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at + (((2 * (piece & 3) + e) ^ (lane & 7)) << 4)), "r"(f[4 * e]), "r"(f[4 * e + 1]), "r"(f[4 * e + 2]), "r"(f[4 * e + 3]) : "memory");
                }
                fence_async_smem();
            };
            auto together = [] { asm volatile("barrier.cta.sync 2, 96;" ::: "memory"); };
            const int r0 = row_of(k_lo), r1 = row_of(k_lo + 64);
            int n0 = row_of(k_lo + 128), n1 = row_of(k_lo + 192);      // the next tile's runs
            if (warp == 0 && lane == 0) {
                bring(kbase, &maps.k, &misc.k_full[0], r0, r1);
                bring(v8base, &maps.v, &misc.v8_full[0], r0, r1);
                if (n > 1) {
                    bring(kbase + kFpCodes, &maps.k, &misc.k_full[1], n0, n1);
                    bring(v8base + kFpCodes, &maps.v, &misc.v8_full[1], n0, n1);
                }
            }
            auto scales_of = [&](int j, int a0, int a1) {      // a tile's runs'
                if (warp == 2 && lane < 2) {
                    const int row = lane ? a1 : a0;
                    misc.scales[j & 3][lane] = row == none ? make_float2(0.f, 0.f) : *reinterpret_cast<const float2*>(a.scales + 2 * (long)(row / ps));
                }
            };
            scales_of(0, r0, r1);
            __syncwarp();
            if (warp == 2 && lane == 0) bar_arrive(smem_u32(&misc.q_full));      // (S of the first tile waits for its scales too)
            for (int j = 0; j < n; j++) {
                const int st = j & 1, k0 = k_lo + j * kFpKeys, l0 = row_of(k0 + 2 * kFpKeys), l1 = row_of(k0 + 2 * kFpKeys + 64);      // (the tile after the next)
                if (j + 1 < n) scales_of(j + 1, n0, n1);      // (S of that tile waits for this one's values)
                if (warp == 0 && lane == 0 && j + 2 < n) {      // (its stage was tile j - 1's)
                    const int kst = (j + 2) % kFpKStages;
                    bar_wait(smem_u32(&misc.k_free[kst]), (((j + 2) / kFpKStages) & 1) ^ 1);
                    bring(kbase + kst * kFpCodes, &maps.k, &misc.k_full[kst], l0, l1);
                }
                __syncwarp();
                bar_wait(smem_u32(&misc.v8_full[st]), (j >> 1) & 1);
                bar_wait(smem_u32(&misc.v_free[st]), ((j >> 1) & 1) ^ 1);
                turn(v8base + st * kFpCodes, vbase + st * kFpTile, k0);
                together();
                if (lane == 0) {
                    bar_arrive(smem_u32(&misc.v_full[st]));
                    if (warp == 0 && j + 2 < n) bring(v8base + st * kFpCodes, &maps.v, &misc.v8_full[st], l0, l1);
                }
                __syncwarp();
                n0 = l0;
                n1 = l1;
            }
        }
    } else {
        // ================================================================ soft-max
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = (warp - 4) >> 2, sp = warp & 3, r = 32 * sp + lane;
        const uint32_t ts = tmem + ((uint32_t)(32 * sp) << 16) + t * 256, to = ts + 128;
        const int tok = t * TOKS + r / RH, h = h0 + r % RH;
        const bool valid = r < TOKS * RH && tok < ntok;
        const int p = pos0 + tok, first = fp8_first_visible(p, a.window, a.chunk);
        float fac;
        {      // the row of Q
            uint32_t w[64];
            const uint4* row = reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.q + ((long)(tok0 + tok) * a.H + h) * 128);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const uint4 v = valid ? row[i] : make_uint4(0, 0, 0, 0);
                w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
            float top = 0.f, odd = 0.f;      // odd: NaN as soon as a value is not finite (e4m3 has no infinity)
#pragma unroll
            for (int i = 0; i < 64; i++) {
                const float x = __uint_as_float(w[i] << 16), y = __uint_as_float(w[i] & 0xffff0000u);
                top = fmaxf(top, fmaxf(fabsf(x), fabsf(y)));
                odd = fmaf(x, 0.f, fmaf(y, 0.f, odd));
            }
            const int up = min(126, max(-120, 7 - ((int)(__float_as_uint(top) >> 23) - 127)));
            const float by = __uint_as_float((uint32_t)(up + 127) << 23);
            fac = valid ? (a.head_scale ? a.scale * a.head_scale[h] : a.scale) / by + odd : 0.f;
            uint8_t* to = smem + t * kFpTile + r * 128;
#pragma unroll
            for (int c = 0; c < 8; c++) {      // 16 columns, both terms
                uint32_t f[4], e[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t u = w[8 * c + 2 * i], v = w[8 * c + 2 * i + 1];
                    const uint2 lo2 = split_e4m3<1>(__uint_as_float(u << 16) * by, __uint_as_float(u & 0xffff0000u) * by), hi2 = split_e4m3<1>(__uint_as_float(v << 16) * by, __uint_as_float(v & 0xffff0000u) * by);
                    f[i] = lo2.x | hi2.x << 16;
                    e[i] = lo2.y | hi2.y << 16;
                }
                *reinterpret_cast<uint4*>(to + ((c ^ (r & 7)) << 4)) = make_uint4(f[0], f[1], f[2], f[3]);
                *reinterpret_cast<uint4*>(to + kFpCodes + ((c ^ (r & 7)) << 4)) = make_uint4(e[0], e[1], e[2], e[3]);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) bar_arrive(smem_u32(&misc.q_full));
        }
        const float softcap = a.softcap, two_over_cap = softcap > 0.f ? 2.0f / softcap : 0.f;
        // scores that are only scaled (by a positive number) go to the exponential as they are
        const bool direct = __all_sync(0xffffffffu, softcap <= 0.f && (fac > 0.f || !valid));
        const int w_tok0 = t * TOKS + 32 * sp / RH, w_tok1 = t * TOKS + min(TOKS - 1, (32 * sp + 31) / RH);      // the warp's first and last token
        const bool w_full = w_tok1 < ntok;
        const int w_last_first = fp8_first_visible(pos0 + w_tok1, a.window, a.chunk);
        float m_ref = -INFINITY, l = 0.f;
        for (int i64 = 0; i64 < 2 * n; i64++) {
            const int k0 = k_lo + 64 * i64, buf = i64 & 1;
            const uint32_t tb = ts + 64 * buf;
            bar_wait(smem_u32(&misc.s_full[t][buf]), (i64 >> 1) & 1);
            tc_fence_after();
            float s[64];
#pragma unroll
            for (int q = 0; q < 2; q++) {
                uint32_t v[32];
                tmem_ld32(tb + 32 * q, v);
#pragma unroll
                for (int i = 0; i < 32; i++) s[32 * q + i] = __uint_as_float(v[i]);
            }
            const float2 sc = misc.scales[(i64 >> 1) & 3][buf];
            const uint32_t vbits = __float_as_uint(sc.y);
            float c = direct ? fmaxf(fac * sc.x * kLog2e, 1.2e-38f) : fac * sc.x;      // (above zero: -inf times it stays that)
            const float ve = (float)((int)(vbits >> 23) - 127), inv = vbits ? __uint_as_float((254u << 23) - vbits) : 0.f;
            tmem_wait_ld();
            // (the loads above are in registers only now)
#pragma unroll
            for (int i = 0; i < 64; i++) asm volatile("" : "+f"(s[i]));
            if (!direct) {
#pragma unroll
                for (int i = 0; i < 64; i++) {
                    float x = s[i] * c;
                    if (softcap > 0.f) x = softcap * (1.0f - __fdividef(2.0f, __expf(x * two_over_cap) + 1.0f));      // c tanh(s / c): a few 1e-7 of the cap off
                    s[i] = x * kLog2e;
                }
                c = 1.f;
            }
            if (!(vbits && w_full && k0 + 64 <= k_hi && k0 + 63 <= pos0 + w_tok0 && k0 >= w_last_first)) {
                const int i0 = first - k0, i1 = valid && vbits ? min(p, k_hi - 1) - k0 : -1;
#pragma unroll
                for (int i = 0; i < 64; i++)
                    if (i < i0 || i > i1) s[i] = -INFINITY;
            }
            float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i < 64; i += 4)
#pragma unroll
                for (int q = 0; q < 4; q++) mx[q] = fmaxf(mx[q], s[i + q]);
            const float m_new = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), c, ve);
            const bool raise = m_new > m_ref + kFmRaise || (m_ref == -INFINITY && m_new > -INFINITY);
            if (__any_sync(0xffffffffu, raise)) {
                const float alpha = raise ? exp2_approx(m_ref - (m_new - kFmTop)) : 1.f;      // (2^-inf = 0: nothing was summed yet)
                if (raise) { m_ref = m_new - kFmTop; l *= alpha; }
                if (i64 > 0) {
                    bar_wait(smem_u32(&misc.pv_done[t][buf ^ 1]), ((i64 - 1) >> 1) & 1);
                    tc_fence_after();
#pragma unroll 1
                    for (int q = 0; q < 4; q++) {
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
            const f32x2 c2 = pack2(c, c), o2 = pack2(ve - u, ve - u);
            f32x2 sum[2] = {0, 0};
            uint32_t pk[32];
#pragma unroll
            for (int i = 0; i < 32; i++) {
                float e0, e1;
                unpack2(fma2(pack2(s[2 * i], s[2 * i + 1]), c2, o2), e0, e1);
                e0 = exp2_approx(e0);
                e1 = exp2_approx(e1);
                pk[i] = pack_f16(e0, e1);
                sum[i & 1] = add2(sum[i & 1], pack2(e0, e1));
            }
            tmem_st32(tb, pk);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(smem_u32(&misc.p_full[t][buf]));
            float a0, a1, a2, a3;
            unpack2(sum[0], a0, a1);
            unpack2(sum[1], a2, a3);
            l = fmaf((a0 + a1) + (a2 + a3), inv, l);
        }
        // the last product of each buffer: its n-th.  (The (n - 1)-th of both are complete, the scores that the loop waited for last are behind them; a barrier for both buffers would stand
        // one phase or two behind what is known, and a wait for a phase that is two back never ends)
        bar_wait(smem_u32(&misc.pv_done[t][0]), (n - 1) & 1);
        bar_wait(smem_u32(&misc.pv_done[t][1]), (n - 1) & 1);
        tc_fence_after();
        const long row = (long)(tok0 + tok) * a.H + h;
        float* part = cut ? a.partial + (row * a.parts + blockIdx.z) * 130 : nullptr;
        float k = 1.f;
        if (cut) {
            if (valid) *reinterpret_cast<float2*>(part) = make_float2(m_ref, l);
        } else {
            if (a.sink) k = fp8_sink(a.sink[h], m_ref, l);
            k = l > 0.f || l != l ? k * a.out_scale / l : 0.f;
        }
        __nv_bfloat16* out = (__nv_bfloat16*)a.out + (long)(tok0 + tok) * a.out_stride + (long)h * 128;
        const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
        const int bad = min(misc.n_bad, kFpBad);
#pragma unroll 1
        for (int q = 0; q < 4; q++) {
            uint32_t v[32];
            tmem_ld32(to + 32 * q, v);
            tmem_wait_ld();
            if (!valid) continue;
            if (bad > 0) {
                const bool whole = misc.n_bad > kFpBad && misc.bad_lo <= p && misc.bad_hi >= first;      // (more than the list holds: rows that see keys between the first and the last)
                for (int b = 0; b < bad; b++) {
                    const int2 e = misc.bad[b];
                    const int run = e.y >> 16;
                    const uint32_t mask = e.x >= first && e.x <= p && (run >> 1) == q ? (uint32_t)(e.y & 0xffff) << (16 * (run & 1)) : 0u;
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (whole || (mask >> i & 1)) v[i] = 0x7fffffffu;
                }
            }
            if (cut) {
#pragma unroll
                for (int i = 0; i < 16; i++) *reinterpret_cast<float2*>(part + 2 + 32 * q + 2 * i) = make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                continue;
            }
            uint32_t o[16];
#pragma unroll
            for (int i = 0; i < 16; i++) o[i] = pack_bf16(__uint_as_float(v[2 * i]) * k, __uint_as_float(v[2 * i + 1]) * k);
            if (vec) {
#pragma unroll
                for (int i = 0; i < 4; i++) *reinterpret_cast<uint4*>(out + 32 * q + 8 * i) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            } else {
#pragma unroll
                for (int i = 0; i < 32; i++) reinterpret_cast<uint16_t*>(out)[32 * q + i] = (uint16_t)(o[i >> 1] >> (16 * (i & 1)));
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

// whether these tiles take the call: portions of half a row tile's tokens on average
static bool fp_takes(const ktb200_fp8_attn_params* c, int n_tokens, int dtype) {
    return fm_takes(c, dtype) && c->dim == 128 && c->vdim == 128 && c->page_size % 64 == 0 && c->n_pages > 0 && (long)c->n_pages * c->kv_heads * c->page_size < (1L << 31) &&
           (long)n_tokens * fm_heads(c->heads / c->kv_heads) >= 64L * c->n_seqs;
}
static int fp_launch(const Fp8Attn& a, int RH, dim3 grid, cudaStream_t s) {
    FdMaps maps;
    const int rc = fd_maps(maps, a, 64);
    if (rc) return rc;
    KTB_CUDA_CHECK(raise_smem_limit((const void*)fp8_attn_prompt_kernel, kFpSmem));
    if (grid.x > 65535) { set_error("fp8_cache_attn: too many tokens"); return KTB200_EINVAL; }
    KTB_CUDA_CHECK(launch_pdl(fp8_attn_prompt_kernel, dim3(grid.y, grid.x, grid.z), dim3(kFpThreads), (size_t)kFpSmem, s, maps, a, RH));
    return KTB200_OK;
}

}  // namespace ktb
