// Keys and values of the expanded form: [k | v] of row r and head h = W_h c_r for the rows that latent_gather_kernel laid side by side (bf16, K = 512).
// Persistent pairs of CTAs (cta_group::2): a pair's tile is 256 rows x one head (bn = nope_dim + vdim columns), each CTA has 128 of the rows and brings half of the head's weight rows, which
// both tensor cores read.
// A head's weights (64 KB to 128 KB a CTA) stay in shared memory while the pair walks the rows: brought again for each tile they were two of four operand bytes, and at 43 bytes a cycle and SM
// from L2 the copies bound the kernel (4049 rows, 128 heads: 120 us).
//     warp 0 TMA: weights of a new head run by run of 64 columns as the last products of the old one are done with them, rows through a ring; a pair's bytes are counted by the first CTA's barriers
//     warp 1 of the first CTA the pair's products; warps 4-7 and 8-11 results, 64 columns at a time through shared memory and out by TMA.  Two accumulators of bn columns.  (Sectors of 32 bytes
//     stored by the threads took 120 us for 4049 rows and 128 heads, so 112: a tile has only 512 columns of products to hide its 64 KB of results behind)
// Tiles stand in one line, rows fastest, cut into equal runs, one a pair.
// Results: [head of the pass][row][bn], rows of the plan (a multiple of 128: a CTA's rows are all there or not at all), one rounding.
#pragma once
#include "latent_attn.cuh"

namespace ktb {

constexpr int kLxThreads = 384, kLxBlocks = kLatent / 64, kLxBox = 128 * 128, kLxStages = 4;      // runs of 64 columns; 128 rows of one; the ring of rows
struct LxMisc {
    unsigned long long w_full[kLxBlocks], w_free[kLxBlocks], full[kLxStages], free[kLxStages], d_full[2], d_free[2];
    uint32_t tmem_base;
};
constexpr int kLxRing = kLxBlocks * kLxBox, kLxOut = kLxRing + kLxStages * kLxBox, kLxRoom = kLxOut + 2 * kLxBox, kLxSmem = kLxRoom + (int)sizeof(LxMisc) + 1024;
static_assert(kLxSmem <= 232448, "shared memory budget");

// a line of `line` tiles in `runs` runs that differ by one tile at most: the first tile of run i, and the run that has tile x
__device__ __forceinline__ int latent_run(int line, int runs, int i) { return line / runs * i + min(i, line % runs); }
__device__ __forceinline__ int latent_run_of(int line, int runs, int x) {
    const int n = line / runs, more = line % runs, long_ones = more * (n + 1);
    return x < long_ones ? x / (n + 1) : more + (x - long_ones) / n;
}
__device__ __forceinline__ void lx_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void lx_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t lx_cluster_at(uint32_t addr, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
    return at;
}
// a box into this CTA's shared memory, counted by a barrier of either CTA of the pair
__device__ __forceinline__ void lx_load_pair(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(m), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
// Four products of the pair on consecutive K-steps of 32 bytes, and the barriers (of both CTAs) that complete when all so far have (0: not asked for); called by a converged warp
__device__ __forceinline__ void lx_mma_pair_x4(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate, uint32_t bar0, uint32_t bar1) {
    asm volatile(
        "{\n"
        ".reg .pred p, q, c, e, t;\n"
        ".reg .b32 r;\n"
        ".reg .b64 a, b;\n"
        ".reg .b16 both;\n"
        "mov.b16 both, 3;\n"
        "elect.sync r|q, 0xffffffff;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "setp.eq.b32 t, %4, %4;\n"
        "setp.ne.and.b32 c, %5, 0, q;\n"
        "setp.ne.and.b32 e, %6, 0, q;\n"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
        "add.u64 a, %1, 2;\n"
        "add.u64 b, %2, 2;\n"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, t;\n"
        "add.u64 a, a, 2;\n"
        "add.u64 b, b, 2;\n"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, t;\n"
        "add.u64 a, a, 2;\n"
        "add.u64 b, b, 2;\n"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, t;\n"
        "@c tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%5], both;\n"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%6], both;\n"
        "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(bar0), "r"(bar1) : "memory");
}

__device__ __forceinline__ void lx_commit_pair(uint32_t bar) {      // both CTAs' barrier completes when all products so far have
    asm volatile(
        "{\n"
        ".reg .pred q;\n"
        ".reg .b32 r;\n"
        ".reg .b16 both;\n"
        "mov.b16 both, 3;\n"
        "elect.sync r|q, 0xffffffff;\n"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], both;\n"
        "}\n" ::"r"(bar)
        : "memory");
}

// lat: rows of [512 | 64] (the first 512 columns are read); wmap: rows of w; out: rows of bn columns, boxes of 128 x 64
__global__ void __launch_bounds__(kLxThreads, 1) __cluster_dims__(2, 1, 1)
    latent_expand_kernel(const __grid_constant__ CUtensorMap lat, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap out, const int* plan, int bn, int heads, int pass) {
    using namespace umma;
    extern __shared__ __align__(16) uint8_t lx_smem_raw[];
    const uint32_t raw = smem_u32(lx_smem_raw), base = (raw + 1023u) & ~1023u;
    LxMisc& misc = *reinterpret_cast<LxMisc*>(lx_smem_raw + (base - raw) + kLxRoom);
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform(tid >> 5), rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    griddep_launch_dependents();
    if (tid == 0) {
        for (int s = 0; s < kLxBlocks; s++) { bar_init(smem_u32(&misc.w_full[s]), 1); bar_init(smem_u32(&misc.w_free[s]), 1); }
        for (int s = 0; s < kLxStages; s++) { bar_init(smem_u32(&misc.full[s]), 1); bar_init(smem_u32(&misc.free[s]), 1); }
        for (int b = 0; b < 2; b++) { bar_init(smem_u32(&misc.d_full[b]), 1); bar_init(smem_u32(&misc.d_free[b]), 16); }
        bar_fence_init();
        tma_prefetch_desc(&lat);
        tma_prefetch_desc(&wmap);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&misc.tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    lx_cluster_arrive();      // (the pair's barriers and tensor memory are there)
    lx_cluster_wait();
    tc_fence_after();
    const uint32_t tmem = uniform(misc.tmem_base);
    griddep_wait();
    const int rows = plan[kPlanRows], h0 = pass * plan[kPlanHeads], nt = min(plan[kPlanHeads], heads - h0), mt = (rows + 255) / 256, line = nt > 0 ? mt * nt : 0;
    const int first = latent_run(line, pairs, pair), end = latent_run(line, pairs, pair + 1);
    if (warp == 0) {
        if (lane == 0 && first < end) {
            int s = 0, ph = 1, h = first / mt, m = first - h * mt, wph = 1;
            for (int tile = first; tile < end; tile++) {
                const bool fresh = tile == first || m == 0;
                for (int kb = 0; kb < kLxBlocks; kb++) {
                    if (fresh) {
                        bar_wait(smem_u32(&misc.w_free[kb]), wph);
                        if (rank == 0) bar_expect_tx(smem_u32(&misc.w_full[kb]), bn * 128);
                        lx_load_pair(base + kb * kLxBox, &wmap, lx_cluster_at(smem_u32(&misc.w_full[kb]), 0), kb * 64, (h0 + h) * bn + rank * (bn / 2));
                    }
                    bar_wait(smem_u32(&misc.free[s]), ph);
                    if (rank == 0) bar_expect_tx(smem_u32(&misc.full[s]), 2 * kLxBox);
                    lx_load_pair(base + kLxRing + s * kLxBox, &lat, lx_cluster_at(smem_u32(&misc.full[s]), 0), kb * 64, m * 256 + rank * 128);
                    if (++s == kLxStages) { s = 0; ph ^= 1; }
                }
                if (fresh) wph ^= 1;
                if (++m == mt) { m = 0; h++; }
            }
        }
        __syncwarp();
    } else if (warp == 1 && rank == 0) {
        const uint32_t idesc = instr_desc(1, 1, 1, 0, 0, 256, 0) | ((uint32_t)(bn >> 3) << 17);
        int s = 0, ph = 0, it = 0, m = first < end ? first % mt : 0, wph = 0;
        for (int tile = first; tile < end; tile++, it++) {
            const int buf = it & 1;
            const bool fresh = tile == first || m == 0, last = tile + 1 == end || m + 1 == mt;      // of this head's
            bar_wait(smem_u32(&misc.d_free[buf]), ((it >> 1) & 1) ^ 1);
            tc_fence_after();
            for (int kb = 0; kb < kLxBlocks; kb++) {
                if (fresh) bar_wait(smem_u32(&misc.w_full[kb]), wph);
                bar_wait(smem_u32(&misc.full[s]), ph);
                tc_fence_after();
                lx_mma_pair_x4(tmem + buf * 256, smem_desc(base + kLxRing + s * kLxBox, 16, 1024, kLayoutSw128), smem_desc(base + kb * kLxBox, 16, 1024, kLayoutSw128), idesc, kb > 0, smem_u32(&misc.free[s]),
                               last ? smem_u32(&misc.w_free[kb]) : 0);
                if (++s == kLxStages) { s = 0; ph ^= 1; }
            }
            lx_commit_pair(smem_u32(&misc.d_full[buf]));
            if (fresh) wph ^= 1;
            if (++m == mt) m = 0;
        }
    } else if (warp >= 4) {
        const int sp = warp & 3, half = (warp - 4) >> 2, r = 32 * sp + lane;
        const bool lead = warp == 4 + 4 * half && lane == 0;      // of the four warps that share a box
        const uint32_t box = base + kLxOut + half * kLxBox;
        int it = 0, h = first < end ? first / mt : 0, m = first < end ? first - h * mt : 0;
        for (int tile = first; tile < end; tile++, it++) {
            const int m0 = m * 256 + rank * 128, row0 = h * rows + m0, buf = it & 1;
            const uint32_t tcol = tmem + ((uint32_t)(32 * sp) << 16) + buf * 256;
            if (++m == mt) { m = 0; h++; }
            bar_wait(smem_u32(&misc.d_full[buf]), (it >> 1) & 1);
            tc_fence_after();
#pragma unroll 1
            for (int c = 64 * half; c < bn; c += 128) {
                uint32_t w[32];
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    uint32_t v[32];
                    tmem_ld32(tcol + c + 32 * q, v);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; i++) w[16 * q + i] = latent_pack(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                }
                if (lead) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // (the box before has left)
                asm volatile("barrier.cta.sync %0, 128;" ::"r"(1 + half) : "memory");
#pragma unroll
                for (int i = 0; i < 8; i++)
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(box + r * 128 + ((i ^ (r & 7)) << 4)), "r"(w[4 * i]), "r"(w[4 * i + 1]), "r"(w[4 * i + 2]), "r"(w[4 * i + 3]) : "memory");
                fence_async_smem();
                asm volatile("barrier.cta.sync %0, 128;" ::"r"(1 + half) : "memory");
                if (lead && m0 < rows) {
                    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(&out), "r"(box), "r"(c), "r"(row0) : "memory");
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(lx_cluster_at(smem_u32(&misc.d_free[buf]), 0)) : "memory");
        }
        if (lead) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    lx_cluster_arrive();      // nobody leaves while the other's copies and products reach for its barriers
    lx_cluster_wait();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

}  // namespace ktb
