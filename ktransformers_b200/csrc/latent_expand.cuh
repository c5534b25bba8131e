// Keys and values of the expanded form: [k | v] of row r and head h = W_h c_r for the rows that latent_gather_kernel laid side by side (bf16, K = 512).
// Persistent pairs of CTAs (cta_group::2): a pair's tile is 256 rows x one head (bn = nope_dim + vdim columns), each CTA has 128 of the rows and brings half of the head's weight rows, which
// both tensor cores read.
//     warp 0 TMA ring (192 KB) of its own half, whose bytes are counted by the first CTA's barriers; warp 1 of the first CTA the pair's products; warps 4-19 results (a thread one row, every
//     fourth run of 16 columns).  Two accumulators of bn columns.
// Tiles run row tile fastest inside groups of kLxGroup, so that the CTAs of a wave share the weight rows and the latents through L2.
// Results: [head of the pass][row][bn], rows of the plan (a multiple of 128: a CTA's rows are all there or not at all), one rounding.
#pragma once
#include "latent_attn.cuh"

namespace ktb {

constexpr int kLxThreads = 640, kLxGroup = 8, kLxRing = 192 * 1024;
struct LxMisc {
    unsigned long long full[8], free[8], d_full[2], d_free[2];
    uint32_t tmem_base;
};
constexpr int kLxSmem = kLxRing + (int)sizeof(LxMisc) + 1024;
static_assert(kLxSmem <= 232448, "shared memory budget");
__host__ __device__ constexpr int lx_stage(int bn) { return 128 * 128 + bn / 2 * 128; }
__host__ __device__ constexpr int lx_stages(int bn) { return kLxRing / lx_stage(bn) < 8 ? kLxRing / lx_stage(bn) : 8; }

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

// lat: rows of [512 | 64] (the first 512 columns are read); wmap: rows of w
__global__ void __launch_bounds__(kLxThreads, 1) __cluster_dims__(2, 1, 1)
    latent_expand_kernel(const __grid_constant__ CUtensorMap lat, const __grid_constant__ CUtensorMap wmap, const int* plan, __nv_bfloat16* out, int bn, int heads, int pass) {
    using namespace umma;
    extern __shared__ __align__(16) uint8_t lx_smem_raw[];
    const uint32_t raw = smem_u32(lx_smem_raw), base = (raw + 1023u) & ~1023u;
    LxMisc& misc = *reinterpret_cast<LxMisc*>(lx_smem_raw + (base - raw) + kLxRing);
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform(tid >> 5), rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int stage = lx_stage(bn), stages = lx_stages(bn);
    constexpr int kBlocks = kLatent / 64;
    griddep_launch_dependents();
    if (tid == 0) {
        for (int s = 0; s < 8; s++) { bar_init(smem_u32(&misc.full[s]), 1); bar_init(smem_u32(&misc.free[s]), 1); }
        for (int b = 0; b < 2; b++) { bar_init(smem_u32(&misc.d_full[b]), 1); bar_init(smem_u32(&misc.d_free[b]), 32); }
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
    const int rows = plan[kPlanRows], h0 = pass * plan[kPlanHeads], nt = min(plan[kPlanHeads], heads - h0), mt = (rows + 255) / 256, tiles = nt > 0 ? mt * nt : 0;
    auto place = [&](int tile, int& m0, int& h) {
        const int per = kLxGroup * nt, g = tile / per, r = tile - g * per, gm = min(kLxGroup, mt - g * kLxGroup);
        h = r / gm;
        m0 = (g * kLxGroup + r % gm) * 256 + rank * 128;
    };
    if (warp == 0) {
        if (lane == 0) {
            int s = 0, ph = 1;
            for (int tile = pair; tile < tiles; tile += pairs) {
                int m0, h;
                place(tile, m0, h);
                for (int kb = 0; kb < kBlocks; kb++) {
                    bar_wait(smem_u32(&misc.free[s]), ph);
                    const uint32_t dst = base + s * stage, bar = lx_cluster_at(smem_u32(&misc.full[s]), 0);
                    if (rank == 0) bar_expect_tx(smem_u32(&misc.full[s]), 2 * stage);
                    lx_load_pair(dst, &lat, bar, kb * 64, m0);
                    lx_load_pair(dst + 128 * 128, &wmap, bar, kb * 64, (h0 + h) * bn + rank * (bn / 2));
                    if (++s == stages) { s = 0; ph ^= 1; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1 && rank == 0) {
        const uint32_t idesc = instr_desc(1, 1, 1, 0, 0, 256, 0) | ((uint32_t)(bn >> 3) << 17);
        int s = 0, ph = 0, it = 0;
        for (int tile = pair; tile < tiles; tile += pairs, it++) {
            const int buf = it & 1;
            bar_wait(smem_u32(&misc.d_free[buf]), ((it >> 1) & 1) ^ 1);
            tc_fence_after();
            for (int kb = 0; kb < kBlocks; kb++) {
                bar_wait(smem_u32(&misc.full[s]), ph);
                tc_fence_after();
                const uint32_t a = base + s * stage, b = a + 128 * 128;
                lx_mma_pair_x4(tmem + buf * 256, smem_desc(a, 16, 1024, kLayoutSw128), smem_desc(b, 16, 1024, kLayoutSw128), idesc, kb > 0, smem_u32(&misc.free[s]),
                               kb + 1 == kBlocks ? smem_u32(&misc.d_full[buf]) : 0);
                if (++s == stages) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp >= 4) {
        const int sp = warp & 3, ch = (warp - 4) >> 2;
        int it = 0;
        for (int tile = pair; tile < tiles; tile += pairs, it++) {
            int m0, h;
            place(tile, m0, h);
            const int buf = it & 1, r = m0 + 32 * sp + lane;
            const uint32_t tcol = tmem + ((uint32_t)(32 * sp) << 16) + buf * 256;
            bar_wait(smem_u32(&misc.d_full[buf]), (it >> 1) & 1);
            tc_fence_after();
            __nv_bfloat16* row = out + ((long)h * rows + r) * bn;
#pragma unroll 1
            for (int c = 16 * ch; c < bn; c += 64) {
                uint32_t v[16];
                tmem_ld16(tcol + c, v);
                tmem_wait_ld();
                if (m0 < rows) {      // (whole sectors of the thread's own row)
                    uint32_t w[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) w[i] = latent_pack(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                    latent_store32(row + c, w);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(lx_cluster_at(smem_u32(&misc.d_free[buf]), 0)) : "memory");
        }
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
