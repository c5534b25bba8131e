// Attention of single tokens over the paged e4m3 cache on tcgen05 (bf16 queries, heads of 128 or 64, pages of whole 16 tokens): the decode step.
//
// A CTA has one token, one key/value head and its query heads, and a part of the key range in tiles of 128 keys.  The codes are operands as they lie in the cache: nothing is converted.
//     S^T = K Q^T     128 keys x N, kind::f8f6f4, K the K-major A operand as TMA delivered it
//     O^T = V^T P^T   128 columns x N, the V tile as an MN-major A operand
// N = 2 RP columns of S^T, NO = 4 RP of O^T, for RP = 8 or 16 heads: what stands against the codes is split into two e4m3 numbers, the second for 16 times what the first leaves.
//   queries   a row moved by a power of two so that its largest stands in [128, 256): exact for bf16 numbers down to 2^-13 of that largest, 2^-21 of it off below
//   weights   p = 2^(t - m), t = s log2(e) + log2(value scale).  Value scales are powers of two: in the exponent they cost nothing and O needs none.  m is 7 below a head's largest t,
//             raised when a t outgrows it by 8.75 (2^8.75 < 448).  The two numbers are within 2^-8 of a weight from 2^-6 on (as a bf16 weight is).  A long context behind one key that has
//             most of the weight lies below that, so a smaller weight stands in two more columns, 2^14 times itself: within 2^-8 of it down to 2^-20, and 2^-28 off below, 2^-35 of the
//             largest.  They are zeros, and not written, as long as a warp has no such weight (64 contexts of 4095 to 8190 keys: 148 us with few, 152 with some in every tile)
// l += p / (value scale), O / l is the result: 2^m drops out.
// Heads of 64 (PAIR = 2): a row of 128 bytes is two neighbouring keys.  Queries and weights then have rows of their own for the first and for the second of a pair, zero where the other's
// columns are; of the products, twice as many as needed, the mixed ones are not looked at.  Bound by the soft-max threads, which write twice the bytes of weights for one of codes: 30 tokens
// over 2000 to 4000 keys, 64 heads over 8, take 45 us (53 with small weights in every tile; the cache's bytes 14) where fp16 mma tiles take 56, one over 60000 keys 25 (29; 9) against 33.
//     warp 0      TMA: K and V tiles, two stages; a tile is runs of 16, 32 or 64 keys, each inside one page (runs that no key of the part lies in come as zeros)
//     warp 1      MMAs: S of the next tile ahead of PV of this one
//     warps 2-5   a thread owns a key: its scores of all heads are one row of S^T, so that scales and masks are its own; maxima are only needed when one has outgrown its
//                 reference, which one barrier with a reduction tells.  At the end a thread owns a column of the result
// A range that is cut for up to eight CTAs is cut evenly, sequence by sequence, and its CTAs are a cluster: each leaves its sums in its shared memory and joins some of the heads from
// all of them, so that there is neither a workspace nor a second launch.  Longer ranges of few sequences go in parts of one length, joined by fp8_merge_kernel.
// TMEM: [S | S | O], N, N and NO columns.  Bound by the cache's bytes: a tile is 32 KB, 740 ns of an SM's share of the memory; three CTAs an SM (two for 16 heads), so that what a CTA
// spends ahead of its first tile and between a tile's steps is another's time.
#pragma once
#include <cuda.h>

#include "umma.cuh"

namespace ktb {

constexpr int kFdThreads = 192, kFdRows = 128, kFdTile = kFdRows * 128, kFdStages = 2;
constexpr float kFdTop = 7.f, kFdRaise = 8.75f;
constexpr float kFdSmall = -6.f, kFdLift = 16384.f, kFdNone = -28.f;      // weights below 2^-6 stand as 2^14 times themselves; those below 2^-28 become zero there
template <int RP> struct FdMisc {
    unsigned long long k_full[kFdStages], k_free[kFdStages], v_full[kFdStages], v_free[kFdStages], s_full[2], s_free[2], p_full[2], p_free[2], q_ready;
    float red[4][RP], fac[RP];
    uint32_t tmem_base;
    int found;
};
// the ring, the queries (2 RP rows, twice for pairs), two buffers of weights (4 RP rows)
template <int RP, int PAIR> constexpr int fd_smem() { return 2 * kFdStages * kFdTile + (2 + 2 * 4) * RP * PAIR * 128 + (int)sizeof(FdMisc<RP>); }
static_assert(3 * (fd_smem<8, 1>() + 1024) <= 228 * 1024, "three CTAs an SM");

struct FdMaps { CUtensorMap k, v; };
constexpr int kFdCluster = 8;
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float cluster_load(uint32_t addr, uint32_t rank) {      // a word of another CTA's shared memory
    uint32_t at;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

// Where the byte of key (column) c of row n of a K-major operand with 128-byte rows and 128-byte swizzle lies
__device__ __forceinline__ uint32_t fd_at(int n, int c) { return (uint32_t)((n >> 3) * 1024 + (n & 7) * 128 + ((((c >> 4) ^ n) & 7) << 4) + (c & 15)); }
__device__ __forceinline__ bool fd_any(bool p) {      // over the four soft-max warps
    uint32_t r;
    asm volatile("{\n.reg .pred a, b;\nsetp.ne.u32 a, %1, 0;\nbarrier.cta.red.or.pred b, 1, 128, a;\nselp.u32 %0, 1, 0, b;\n}" : "=r"(r) : "r"((uint32_t)p) : "memory");
    return r != 0;
}
__device__ __forceinline__ void fd_sync() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }

template <int RP, int PAIR> __global__ void __launch_bounds__(kFdThreads, RP * PAIR == 8 ? 3 : 2) fp8_attn_decode_kernel(const __grid_constant__ FdMaps maps, const Fp8Attn a, int RH, int run) {
    using namespace umma;
    constexpr int N = 2 * RP * PAIR, NO = 2 * N, QP = N * 128, OP = NO * 128, D = 128 / PAIR, KEYS = kFdRows * PAIR;      // QP, OP: bytes of the queries and of a buffer of weights
    extern __shared__ __align__(1024) uint8_t fd_smem_raw[];
    const uint32_t raw = smem_u32(fd_smem_raw), base = (raw + 1023u) & ~1023u;      // (the same number; with raw itself, whose value is known, a call over 1500 keys took 9.6 us, and takes 9.1)
    uint8_t* smem = fd_smem_raw + (base - raw);
    const uint32_t kbase = base, vbase = base + kFdStages * kFdTile, qbase = base + 2 * kFdStages * kFdTile, pbase = qbase + QP;
    FdMisc<RP>& misc = *reinterpret_cast<FdMisc<RP>*>(smem + 2 * kFdStages * kFdTile + QP + 2 * OP);
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform(tid >> 5), ps = a.pages.page_size;
    griddep_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < kFdStages; i++) { bar_init(smem_u32(&misc.k_full[i]), 1); bar_init(smem_u32(&misc.k_free[i]), 1); bar_init(smem_u32(&misc.v_full[i]), 1); bar_init(smem_u32(&misc.v_free[i]), 1); }
        for (int i = 0; i < 2; i++) { bar_init(smem_u32(&misc.s_full[i]), 1); bar_init(smem_u32(&misc.s_free[i]), 4); bar_init(smem_u32(&misc.p_full[i]), 4); bar_init(smem_u32(&misc.p_free[i]), 1); }
        bar_init(smem_u32(&misc.q_ready), 4);
        bar_fence_init();
        tma_prefetch_desc(&maps.k);
        tma_prefetch_desc(&maps.v);
    }
    griddep_wait();
    // What a CTA needs ahead of its first copy, loaded side by side: the token's position and table row, whether a portion has the token, and the token's queries
    const int t = blockIdx.x, R = a.H / a.G, hblocks = R / RH, g = blockIdx.y / hblocks, h0 = g * R + (blockIdx.y % hblocks) * RH;
    const int p = a.pos[t], slot = a.slot[t];
    uint2 q_row[RP / 4];
    if (warp >= 2) {      // a warp a head: a lane has columns 4 lane .. (2 lane ..)
#pragma unroll
        for (int i = 0; i < RP / 4; i++) {
            const int h = warp - 2 + 4 * i;
            const __nv_bfloat16* row = (const __nv_bfloat16*)a.q + ((long)t * a.H + h0 + h) * D + 4 / PAIR * lane;
            q_row[i] = h >= RH ? make_uint2(0, 0) : PAIR == 1 ? *reinterpret_cast<const uint2*>(row) : make_uint2(*reinterpret_cast<const uint32_t*>(row), 0);
        }
    } else if (warp == 0) {
        bool mine = false;
        for (int s = lane; s < a.n_seqs; s += 32) {
            const int start = a.seqs[s], len = a.seqs[a.seqs_stride + s];
            mine |= start >= 0 && start <= a.n_tokens - len && t >= start && t - start < len;
        }
        const bool found = __any_sync(0xffffffffu, mine);
        if (lane == 0) misc.found = found && p >= 0;
    }
    __syncthreads();
    if (!misc.found) return;
    const int lo = fp8_first_visible(p, a.window, a.chunk), lo_al = lo & ~(a.align - 1);
    const int even = a.even, part = even ? ((p + 1 - lo_al + KEYS - 1) / KEYS + even - 1) / even * KEYS : a.part;
    const bool cut = !even && part > 0 && p + 1 - lo_al > part;
    const int k_lo = lo_al + blockIdx.z * part, k_hi = cut || even ? min(p + 1, k_lo + part) : p + 1;
    float* join = reinterpret_cast<float*>(smem);      // a cluster's CTA: (reference, sum) of RP heads, then RP rows of 128 columns, over the ring
    if (k_lo >= k_hi) {
        if (even) {      // nothing to add: the cluster's barriers only
            cluster_arrive();
            cluster_wait();
            cluster_arrive();
            cluster_wait();
        }
        return;
    }
    const int tiles = (k_hi - k_lo + KEYS - 1) / KEYS;
    if (warp == 1) tmem_alloc(smem_u32(&misc.tmem_base), 128);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(misc.tmem_base), tmem_o = tmem + 2 * N;
    const bool slot_ok = (unsigned)slot < (unsigned)a.pages.slots;
    const int* pt = a.pages.table + (slot_ok ? (long)slot * a.pages.max_pages : 0);
    auto page_of = [&](int key) {      // -1: not there
        const int page = pt[(key / ps) % a.pages.max_pages];
        return (unsigned)page < (unsigned)a.pages.n_pages ? page : -1;
    };

    if (warp == 0) {
        // ================================================================ copies
        const int runs = kFdRows / run, ahead = 32 / runs, none = a.pages.n_pages * a.G * (ps / PAIR);      // (rows from `none` on are outside the maps: zeros)
        int row = none;
        for (int j = 0; j < tiles; j++) {
            if (j % ahead == 0) {      // a lane looks one run's page up, for as many tiles as the lanes reach
                const int kp = k_lo + j * KEYS + lane * run * PAIR, page = slot_ok && kp < k_hi && kp + run * PAIR > lo ? page_of(kp) : -1;
                row = page < 0 ? none : (page * a.G + g) * (ps / PAIR) + kp % ps / PAIR;
            }
            const int st = j % kFdStages, ph = ((j / kFdStages) & 1) ^ 1;
            const uint32_t kf = smem_u32(&misc.k_full[st]), vf = smem_u32(&misc.v_full[st]);
            if (lane == 0) {
                bar_wait(smem_u32(&misc.k_free[st]), ph);
                bar_expect_tx(kf, kFdTile);
            }
            for (int i = 0; i < runs; i++) {
                const int r = __shfl_sync(0xffffffffu, row, (j % ahead) * runs + i);
                if (lane == 0) tma_load_2d(kbase + st * kFdTile + i * run * 128, &maps.k, kf, 0, r);
            }
            if (lane == 0) {
                bar_wait(smem_u32(&misc.v_free[st]), ph);
                bar_expect_tx(vf, kFdTile);
            }
            for (int i = 0; i < runs; i++) {
                const int r = __shfl_sync(0xffffffffu, row, (j % ahead) * runs + i);
                if (lane == 0) tma_load_2d(vbase + st * kFdTile + i * run * 128, &maps.v, vf, 0, r);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ================================================================ products (converged warp)
        constexpr uint32_t idesc_s = instr_desc(1, 0, 0, 0, 0, 128, N), idesc_o = instr_desc(1, 0, 0, 1, 0, 128, NO);
        bar_wait(smem_u32(&misc.q_ready), 0);
        for (int j = 0; j <= tiles; j++) {
            if (j < tiles) {
                const int st = j % kFdStages, buf = j & 1;
                bar_wait(smem_u32(&misc.k_full[st]), (j / kFdStages) & 1);
                const int k0 = k_lo + j * KEYS;
                if (PAIR == 2 && (k0 < lo || k0 + KEYS > k_hi)) {      // the first and last tiles: a key that is not seen may be anything, and stands in a row with one that is (0 x NaN)
                    for (int i = lane; i < kFdRows * 8; i += 32) {
                        const int row = i >> 3, c = i & 7, key = k0 + 2 * row + (c >> 2);
                        if (key < lo || key >= k_hi) *reinterpret_cast<uint4*>(smem + (kbase - base) + st * kFdTile + row * 128 + ((c ^ (row & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                    }
                    fence_async_smem();
                    __syncwarp();
                }
                bar_wait(smem_u32(&misc.s_free[buf]), ((j >> 1) & 1) ^ 1);
                tc_fence_after();
                mma_f8_x4(tmem + buf * N, smem_desc(kbase + st * kFdTile, 16, 1024, kLayoutSw128), smem_desc(qbase, 16, 1024, kLayoutSw128), idesc_s, 0, smem_u32(&misc.s_full[buf]),
                          smem_u32(&misc.k_free[st]));
            }
            if (j > 0) {
                const int i = j - 1, st = i % kFdStages, buf = i & 1;
                bar_wait(smem_u32(&misc.v_full[st]), (i / kFdStages) & 1);
                bar_wait(smem_u32(&misc.p_full[buf]), (i >> 1) & 1);
                tc_fence_after();
                // 32 keys a step: 32 rows of V, 32 bytes of P's rows
                mma_f8_x4<256, 2>(tmem_o, smem_desc(vbase + st * kFdTile, 16, 1024, kLayoutSw128), smem_desc(pbase + buf * OP, 16, 1024, kLayoutSw128), idesc_o, i > 0, smem_u32(&misc.p_free[buf]),
                                  smem_u32(&misc.v_free[st]));
            }
        }
    } else {
        // ================================================================ queries, soft-max, result
        const int sp = warp & 3, r = 32 * sp + lane, w4 = warp - 2;
        const uint32_t lanes = (uint32_t)(32 * sp) << 16;
        {
#pragma unroll
            for (int i = 0; i < RP / 4; i++) {
                const int h = w4 + 4 * i;
                const uint2 v = q_row[i];
                const float x[4] = {__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u)};
                float odd = 0.f;
                float top = 0.f;
#pragma unroll
                for (int k = 0; k < 4; k++) { top = fmaxf(top, fabsf(x[k])); odd = fmaf(x[k], 0.f, odd); }
                top = warp_max(top);
                odd = warp_sum(odd);      // NaN where a value is not finite (e4m3 has no infinity)
                const int up = min(126, max(-120, 7 - ((int)(__float_as_uint(top) >> 23) - 127)));      // 2^(7 - e) of a largest 1.f 2^e, within what fp32 holds with its inverse
                const float by = __uint_as_float((uint32_t)(up + 127) << 23);
                const uint2 lo2 = split_e4m3(x[0] * by, x[1] * by), hi2 = split_e4m3(x[2] * by, x[3] * by);
                uint8_t* Q = smem + (qbase - base);
                if constexpr (PAIR == 1) {
                    *reinterpret_cast<uint32_t*>(Q + fd_at(h, 4 * lane)) = lo2.x | hi2.x << 16;
                    *reinterpret_cast<uint32_t*>(Q + fd_at(RP + h, 4 * lane)) = lo2.y | hi2.y << 16;
                } else {
#pragma unroll
                    for (int u = 0; u < 2; u++)
#pragma unroll
                        for (int k = 0; k < 2; k++) {      // row 2 RP u + h (+ RP): key u of a pair
                            *reinterpret_cast<uint16_t*>(Q + fd_at(2 * RP * u + h, 64 * k + 2 * lane)) = u == k ? (uint16_t)lo2.x : (uint16_t)0;
                            *reinterpret_cast<uint16_t*>(Q + fd_at(2 * RP * u + RP + h, 64 * k + 2 * lane)) = u == k ? (uint16_t)lo2.y : (uint16_t)0;
                        }
                }
                if (lane == 0) misc.fac[h] = h < RH ? (a.head_scale ? a.scale * a.head_scale[h0 + h] : a.scale) / by * (a.softcap > 0.f ? 1.f : kLog2e) + odd : 0.f;
            }
            for (int i = tid - 64; i < 2 * PAIR * 2 * RP * 8; i += 128)      // no small weights: rows 2 RP .. 4 RP - 1 (of either key of pairs)
                *reinterpret_cast<uint4*>(smem + (pbase - base) + (2 * (i / (16 * RP)) + 1) * 2 * RP * 128 + i % (16 * RP) * 16) = make_uint4(0, 0, 0, 0);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) bar_arrive(smem_u32(&misc.q_ready));
            fd_sync();      // (the factors and the zeros)
        }
        float fac[RP], m[RP], l[RP];
#pragma unroll
        for (int h = 0; h < RP; h++) { fac[h] = misc.fac[h]; m[h] = -INFINITY; l[h] = 0.f; }
        const float two_over_cap = a.softcap > 0.f ? 2.0f / a.softcap : 0.f, cap = a.softcap * kLog2e;
        // the scales of the thread's keys (which share a page), a tile ahead, and their page, two ahead
        auto look = [&](int j) { const int key = k_lo + j * KEYS + PAIR * r; return slot_ok && key + PAIR > lo && key < k_hi ? page_of(key) : -1; };
        auto scales_of = [&](int page) { return page < 0 ? make_float2(0.f, 0.f) : *reinterpret_cast<const float2*>(a.scales + 2 * ((long)page * a.G + g)); };
        float2 sc = scales_of(look(0));
        int page1 = look(1);
        uint32_t lifted = 0;      // the buffers whose columns of small weights this warp has written
        for (int j = 0; j < tiles; j++) {
            const int buf = j & 1;
            const float2 next = scales_of(page1);
            page1 = look(j + 2);
            const int key0 = k_lo + j * KEYS + PAIR * r;
            const bool there = sc.y > 0.f;      // (scales of keys that are not seen are zero)
            bar_wait(smem_u32(&misc.s_full[buf]), (j >> 1) & 1);
            tc_fence_after();
            uint32_t s[N];
            if constexpr (N == 16) tmem_ld16(tmem + lanes + buf * N, s); else tmem_ld32(tmem + lanes + buf * N, s);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(smem_u32(&misc.s_free[buf]));
            const float ve = (float)((int)(__float_as_uint(sc.y) >> 23) - 127), inv = there ? __uint_as_float((254u << 23) - __float_as_uint(sc.y)) : 0.f;
            float x[PAIR * RP];
            bool up = false;
#pragma unroll
            for (int i = 0; i < PAIR * RP; i++) {
                const int u = i / RP, h = i % RP;
                x[i] = fmaf(__uint_as_float(s[2 * RP * u + RP + h]), 0.0625f, __uint_as_float(s[2 * RP * u + h])) * (fac[h] * sc.x);
            }
            if (a.softcap > 0.f) {
#pragma unroll
                for (int i = 0; i < PAIR * RP; i++) x[i] = cap * (1.0f - __fdividef(2.0f, __expf(x[i] * two_over_cap) + 1.0f));      // c tanh(s / c): a few 1e-7 of the cap off
            }
#pragma unroll
            for (int i = 0; i < PAIR * RP; i++) {
                x[i] = there && key0 + i / RP >= lo && key0 + i / RP < k_hi ? x[i] + ve : -INFINITY;
                up |= x[i] > m[i % RP] + kFdRaise;
            }
            if (fd_any(up)) {      // (always in the first tile that has a key)
#pragma unroll
                for (int h = 0; h < RP; h++) {
                    const float top = warp_max(PAIR == 1 ? x[h] : fmaxf(x[h], x[PAIR * RP - RP + h]));
                    if (lane == 0) misc.red[w4][h] = top;
                }
                fd_sync();
                float k[RP];
#pragma unroll
                for (int h = 0; h < RP; h++) {
                    const float top = fmaxf(fmaxf(misc.red[0][h], misc.red[1][h]), fmaxf(misc.red[2][h], misc.red[3][h]));
                    k[h] = 1.f;
                    if (top > m[h] + kFdRaise) {
                        k[h] = exp2_approx(m[h] - (top - kFdTop));      // (2^-inf = 0: nothing was summed yet)
                        m[h] = top - kFdTop;
                        l[h] *= k[h];
                    }
                }
                if (j > 0) {
                    bar_wait(smem_u32(&misc.p_free[buf ^ 1]), ((j - 1) >> 1) & 1);      // PV of the tile before this one is complete
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < NO; c += 32) {
                        uint32_t o[32];
                        tmem_ld32(tmem_o + lanes + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * k[i % RP]);
                        tmem_st32(tmem_o + lanes + c, o);
                    }
                    tmem_wait_st();
                    tc_fence_before();
                }
            }
            if (j > 1) bar_wait(smem_u32(&misc.p_free[buf]), ((j - 2) >> 1) & 1);
            bool small = false;
#pragma unroll
            for (int i = 0; i < PAIR * RP; i++) {
                x[i] -= m[i % RP] == -INFINITY ? 0.f : m[i % RP];
                small |= x[i] < kFdSmall && x[i] > kFdNone;
            }
            small = __any_sync(0xffffffffu, small);
            const bool wide = small || (lifted >> buf & 1);      // (what the warp wrote there two tiles ago is taken back)
            uint8_t* P = smem + (pbase - base) + buf * OP;
            auto put = [&](int n, float p0, float p1) {      // rows n, n + 1 of both terms
                const uint2 c = split_e4m3(p0, p1);
                P[fd_at(n, r)] = (uint8_t)c.x;
                P[fd_at(n + 1, r)] = (uint8_t)(c.x >> 8);
                P[fd_at(n + RP, r)] = (uint8_t)c.y;
                P[fd_at(n + RP + 1, r)] = (uint8_t)(c.y >> 8);
            };
#pragma unroll
            for (int i = 0; i < PAIR * RP; i += 2) {
                const int h = i % RP, n = i / RP * 4 * RP + h;
                float p0 = exp2_approx(x[i]), p1 = exp2_approx(x[i + 1]);
                l[h] = fmaf(p0, inv, l[h]);
                l[h + 1] = fmaf(p1, inv, l[h + 1]);
                if (wide) {
                    const bool s0 = x[i] < kFdSmall, s1 = x[i + 1] < kFdSmall;
                    put(n + 2 * RP, s0 ? p0 * kFdLift : 0.f, s1 ? p1 * kFdLift : 0.f);
                    p0 = s0 ? 0.f : p0;
                    p1 = s1 ? 0.f : p1;
                }
                put(n, p0, p1);
            }
            lifted = (lifted & ~(1u << buf)) | (uint32_t)small << buf;
            const int k0 = k_lo + j * KEYS;
            if (k0 < lo || k0 + KEYS > k_hi) {      // the first and last tiles: values of keys that are not seen may be anything (0 x NaN)
                const int st = j % kFdStages;
                bar_wait(smem_u32(&misc.v_full[st]), (j / kFdStages) & 1);
#pragma unroll
                for (int u = 0; u < PAIR; u++)
                    if (key0 + u < lo || key0 + u >= k_hi) {
#pragma unroll
                        for (int i = 0; i < 8 / PAIR; i++)
                            *reinterpret_cast<uint4*>(smem + (vbase - base) + st * kFdTile + r * 128 + (((8 / PAIR * u + i) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                    }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) bar_arrive(smem_u32(&misc.p_full[buf]));
            sc = next;
        }
        // sums over the keys' threads (the last tile's maxima have been read by all)
        fd_sync();
#pragma unroll
        for (int h = 0; h < RP; h++) {
            const float sum = warp_sum(l[h]);
            if (lane == 0) misc.red[w4][h] = sum;
        }
        bar_wait(smem_u32(&misc.p_free[(tiles - 1) & 1]), ((tiles - 1) >> 1) & 1);
        tc_fence_after();
        float v[RP];      // of column r; heads of 64: what the first keys of pairs give it, and from thread r + 64 what the second ones do
#pragma unroll
        for (int h = 0; h < RP; h++) v[h] = 0.f;
#pragma unroll
        for (int c = 4 * RP - 32; c >= 0; c -= 32) {      // small weights first
            uint32_t o[32];
            tmem_ld32(tmem_o + lanes + (PAIR == 2 && sp >= 2 ? 4 * RP : 0) + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 31; i >= 0; i--) {
                const int term = (c + i) / RP;
                v[i % RP] = fmaf(__uint_as_float(o[i]), (term & 1 ? 0.0625f : 1.f) * (term & 2 ? 1.f / kFdLift : 1.f), v[i % RP]);
            }
        }
        if constexpr (PAIR == 2) {
            float* other = join + 2 * RP + 128 * RP;
            if (r >= 64) {
#pragma unroll
                for (int h = 0; h < RP; h++) other[64 * h + r - 64] = v[h];
            }
            fd_sync();
            if (r < 64) {
#pragma unroll
                for (int h = 0; h < RP; h++) v[h] += other[64 * h + r];
            }
        }
        fd_sync();
#pragma unroll
        for (int h = 0; h < RP; h++) {
            if (h >= RH || r >= D) break;
            float sum = (misc.red[0][h] + misc.red[1][h]) + (misc.red[2][h] + misc.red[3][h]);
            const long row = (long)t * a.H + h0 + h;
            if (even) {
                if (r == 0) { join[2 * h] = m[h]; join[2 * h + 1] = sum; }
                join[2 * RP + 128 * h + r] = v[h];
            } else if (cut) {
                float* part = a.partial + (row * a.parts + blockIdx.z) * (D + 2);
                if (r == 0) { part[0] = m[h]; part[1] = sum; }
                part[2 + r] = v[h];
            } else {
                if (a.sink) v[h] *= fp8_sink(a.sink[h0 + h], m[h], sum);
                ((__nv_bfloat16*)a.out)[(long)t * a.out_stride + (long)(h0 + h) * D + r] = __float2bfloat16_rn(sum > 0.f || sum != sum ? v[h] * (a.out_scale / sum) : 0.f);
            }
        }
    }
    tc_fence_before();
    if (even) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (warp >= 2) {
            const int c = tid - 64, cuts = (p + 1 - lo_al + part - 1) / part;      // the CTAs that have keys
            for (int h = blockIdx.z; h < RH && c < D; h += cuts) {
                const float sink = a.sink ? a.sink[h0 + h] * kLog2e : -INFINITY;
                float mk[kFdCluster], lk[kFdCluster], vk[kFdCluster], top = sink;
#pragma unroll
                for (int k = 0; k < kFdCluster; k++)
                    if (k < cuts) {
                        mk[k] = cluster_load(base + 8 * h, k);
                        lk[k] = cluster_load(base + 8 * h + 4, k);
                        vk[k] = mk[k] > -INFINITY ? cluster_load(base + 8 * RP + 512 * h + 4 * c, k) : 0.f;
                        top = fmaxf(top, mk[k]);
                    }
                float sum = !a.sink ? 0.f : sink == top ? 1.f : exp2_approx(sink - top), v = 0.f;
#pragma unroll
                for (int k = 0; k < kFdCluster; k++)
                    if (k < cuts) {
                        const float w = mk[k] > -INFINITY ? exp2_approx(mk[k] - top) : lk[k];      // (nothing seen: 0; scores of NaN have a sum of NaN and no reference)
                        sum = fmaf(lk[k], mk[k] > -INFINITY ? w : 1.f, sum);
                        v = fmaf(vk[k], w, v);
                    }
                v = sum > 0.f || sum != sum ? v * (a.out_scale / sum) : 0.f;
                ((__nv_bfloat16*)a.out)[(long)t * a.out_stride + (long)(h0 + h) * D + c] = __float2bfloat16_rn(v);
            }
        }
        __syncwarp();
        cluster_arrive();      // nobody leaves while its shared memory is read
        cluster_wait();
    } else {
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 128);
    }
}

static bool fd_takes(const ktb200_fp8_attn_params* c, int n_tokens, int dtype) {
    return fm_takes(c, dtype) && c->dim == c->vdim && (c->dim == 128 || c->dim == 64) && c->page_size % 16 == 0 && (long)n_tokens <= 2L * c->n_seqs &&
           (long)c->n_pages * c->kv_heads * c->page_size < (1L << 31) && c->n_pages > 0;
}
// heads of a group that one CTA takes: 16 at most, 8 for heads of 64
static int fd_heads(int R, int dim) {
    int h = fm_heads(R);
    if (dim == 64 && h > 8)
        for (h = 8; R % h; h--) {}
    return h;
}
template <int RP, int PAIR> static cudaError_t fd_launch_as(const FdMaps& maps, const Fp8Attn& a, int RH, int run, dim3 grid, cudaStream_t s) {
    const cudaError_t e = raise_smem_limit((const void*)fp8_attn_decode_kernel<RP, PAIR>, fd_smem<RP, PAIR>());
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t lc{};
    lc.gridDim = grid; lc.blockDim = dim3(kFdThreads); lc.dynamicSmemBytes = fd_smem<RP, PAIR>(); lc.stream = s;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (pdl_enabled()) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (a.even) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = 1; at[n].val.clusterDim.y = 1; at[n++].val.clusterDim.z = a.even;
    }
    lc.attrs = at;
    lc.numAttrs = n;
    return cudaLaunchKernelEx(&lc, fp8_attn_decode_kernel<RP, PAIR>, maps, a, RH, run);
}
// the codes as rows of 128 bytes, boxes of `run` rows, 128-byte-swizzled
static int fd_maps(FdMaps& maps, const Fp8Attn& a, int run) {
    const umma::EncodeTiledFn enc = umma::encode_tiled();
    if (!enc) { set_error("fp8_cache_attn: cuTensorMapEncodeTiled is not available from this driver"); return KTB200_ECUDA; }
    const cuuint64_t dims[2] = {128, (cuuint64_t)a.pages.n_pages * a.G * a.pages.page_size * a.d / 128}, strides[1] = {128};
    const cuuint32_t box[2] = {128, (cuuint32_t)run}, estr[2] = {1, 1};
    for (int i = 0; i < 2; i++) {
        const CUresult cr = enc(i ? &maps.v : &maps.k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(i ? a.v_codes : a.k_codes), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (cr != CUDA_SUCCESS) { set_error("fp8_cache_attn: cuTensorMapEncodeTiled failed (%d)", (int)cr); return KTB200_ECUDA; }
    }
    return KTB200_OK;
}
static int fd_launch(const Fp8Attn& a, int RH, dim3 grid, cudaStream_t s) {
    const int pair = 128 / a.d;
    int run = 64;      // rows of a box: whole boxes in a page
    while (a.pages.page_size % (run * pair)) run >>= 1;
    FdMaps maps;
    const int rc = fd_maps(maps, a, run);
    if (rc) return rc;
    const auto launch = pair == 2 ? fd_launch_as<8, 2> : RH <= 8 ? fd_launch_as<8, 1> : fd_launch_as<16, 1>;
    KTB_CUDA_CHECK(launch(maps, a, RH, run, grid, s));
    return KTB200_OK;
}

}  // namespace ktb
