// Absorbed attention on pairs of CTAs (cta_group::2): queries that absorb_kernel has brought to the latents, keys and values the latents themselves.
//     s = [q' | q_rot] . [c | k_rot] scale,  o' = sum p c / sum p
// A pair's block is 128 consecutive rows = (token, head) of one portion, 64 a CTA; keys run in tiles of 128.  M = 128 of a pair puts a CTA's 64 rows on all 128 lanes of its tensor memory, half of
// the columns on the upper 64, so that O [64][512] fits (256 columns) and products of N = 256 run at the full rate (64 cycles; one CTA with 64 rows has half of it).
//     S = Q K^T       N = 128 keys, of which a CTA brings its 64 (all 576 columns)
//     O += P V        N = 256 columns twice, of which a CTA brings 128 (all 128 keys): 36 x 41 + 16 x 64 cycles a tile
//     warp 0 TMA, block by block: what a product is done with is loaded again for the next tile, so that one stage of each is enough (a block has a tile's time to come)
//     warp 1 of the first CTA the products, S of the next tile ahead of the values of this one
//     warps 2-5 soft-max: a thread owns a row and half of the tile's keys; P (bf16, each weight 2^-9 of itself off) goes to shared memory.  The running maximum is raised, and O scaled, only when a
//     tile's outgrows it by 2^8
// All tiles of all blocks stand in one line that is cut into equal runs, one a pair; blocks that are cut leave fp32 parts for latent_few_merge_kernel, whole ones are done.
// Tiles that not all rows see whole, or whose last rows are not there, come from `tails`: copies with zeros for what is not there or not finite, and bits that say so (latent_few_prep_kernel).
// Pages of whole tiles that are not there are zeros too; a tile's are looked up only where prep found a portion with some (always: 32 decoded tokens 104 us, now 101).
// Bound by its copies beside the products: 278 KB a pair and tile (45 tokens behind 30000 keys: 2.96 GB from L2 in 325 us, 9.1 TB/s, tensor pipe 59 % active; 32 decoded tokens: 457 MB in 81 us with
// 242 MB of them from memory, 34 %).  Keys' tiles in L2 ahead of their use did not help (341 -> 358).
// Shared memory: queries 72 KB, keys 72, values 64, weights 16.  TMEM: O 256 columns, S two buffers of 64.
#pragma once
#include "latent_attn.cuh"
#include "latent_expand.cuh"

namespace ktb {

constexpr int kFewThreads = 192, kFewBox = 8192, kFewRows = 128, kFewK = 9, kFewTile = 128;      // bytes of 64 rows x 64 columns; rows of a block; runs of 64 key columns
constexpr int kFewOffK = kFewK * kFewBox, kFewOffV = kFewOffK + kFewK * kFewBox, kFewOffP = kFewOffV + 8 * kFewBox, kFewRoom = kFewOffP + 2 * kFewBox;
struct FewMisc {
    unsigned long long q_full, q_free, k_full[kFewK], k_free[kFewK], v_full[4], v_free[4], s_full[2], p_full, pv_done, o_free;
    uint32_t tmem_base;
    float top[2][2][64];      // [tile][half of the keys][row]
};
constexpr int kFewSmem = kFewRoom + (int)sizeof(FewMisc) + 1024;
static_assert(kFewSmem <= 232448, "shared memory budget");

struct __align__(16) FewBlock {
    int row0, rows, lead, seq;      // first row of q'; rows; rows of the portion ahead of it; its portion
    int pos0, tile0, tiles, tail;   // that one's first position; its first tile in the line, its tiles, its portion's first among the tails
    int run0, parts, late, whole;   // the run that has its first tile, the runs that have one; whether that run has tiles of another block before them; its portion's tiles that all rows see whole
};
// what latent_few_prep_kernel leaves: ints tiles of the line, blocks, pairs that have a run (of kFewRun tiles and more), then (from 4 on) for each its first block and tile in it, then FewBlock
// from few_blocks_at
constexpr int kFewLine = 0, kFewBlocks = 1, kFewRuns = 2, kFewPairs = 4, kFewRun = 2;
__host__ __device__ inline long few_blocks_at(int pairs) { return (kFewPairs + 2L * pairs + 3) / 4 * 4; }
struct LatentFew {
    ktb200_latent_attn_params p;
    int* plan;
    int n_tokens, block_cap, tail_cap, pairs, box;        // room for blocks and tails; rows of a copy: 64 or 32
    const int* rows_plan;                                 // rows side by side (latent_plan_kernel): no tails
    const uint32_t *bad, *gone;                           // a bit a row of those, or of the tails: who sees it is NaN; nobody sees it
    const uint4* holes;                                   // for each tile of the tails: of its portion's first, whether pages ahead of it are not there
    float scale_log2;
    __nv_bfloat16* sums;                                  // [T][heads][512]
    float *o_part, *ml_part;                              // [2 pairs][128][512], [2 pairs][128][2]
};

__device__ __forceinline__ int few_whole(const LatentPortion& q) { return min(q.pos, q.end - 1) / kFewTile; }      // (at least one tile is behind them)
__device__ __forceinline__ int few_tails(const LatentPortion& q) { return q.count > 0 ? (q.end + kFewTile - 1) / kFewTile - few_whole(q) : 0; }

// CTA 0: blocks, the line, its cuts.  The others: 32 rows of the tails each
__global__ void __launch_bounds__(256) latent_few_prep_kernel(const LatentFew a, __nv_bfloat16* tails, uint32_t* tail_bad, uint32_t* tail_gone, uint32_t* tail_holes) {
    const ktb200_latent_attn_params& p = a.p;
    griddep_wait();
    griddep_launch_dependents();      // (behind the wait: the next kernels' weights then wait for nothing)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, H = p.heads;
    __shared__ int sums[8], carry[3];
    __shared__ uint32_t odd[8][2];
    if (blockIdx.x > 0) {
        const int g = blockIdx.x - 1, tile = g / 4;
        int seq = -1, at = 0, before = 0;
        LatentPortion q{};
        for (int s0 = 0; s0 < p.n_seqs; s0 += 32) {
            const LatentPortion mine = s0 + lane < p.n_seqs ? latent_portion(p, a.n_tokens, s0 + lane) : LatentPortion{};
            const int n = few_tails(mine);
            int sum = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
            }
            const unsigned has = __ballot_sync(0xffffffffu, tile < before + sum);
            if (has) {
                const int l = __ffs(has) - 1;
                seq = s0 + l;
                at = tile - (before + __shfl_sync(0xffffffffu, sum - n, l));
                q = LatentPortion{__shfl_sync(0xffffffffu, mine.first, l), __shfl_sync(0xffffffffu, mine.count, l), __shfl_sync(0xffffffffu, mine.pos, l), __shfl_sync(0xffffffffu, mine.slot, l), __shfl_sync(0xffffffffu, mine.end, l)};
                break;
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (seq < 0) return;
        const int key0 = (few_whole(q) + at) * kFewTile + (g & 3) * 32, keys = q.end;
        uint32_t mine = 0, lost = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int key = key0 + 4 * warp + i;
            int page = -1;
            if (key < keys) page = p.page_table[(long)q.slot * p.max_pages + key / p.page_size];
            const bool there = (unsigned)page < (unsigned)p.n_pages;
            if (key < keys && !there) lost |= 1u << (4 * warp + i);
            if (latent_copy_row((const __nv_bfloat16*)p.cache + ((long)page * p.page_size + key % p.page_size) * kLatentRow, there, tails + ((long)g * 32 + 4 * warp + i) * kLatentRow, true)) mine |= 1u << (4 * warp + i);
        }
        if (lane == 0) { odd[warp][0] = mine; odd[warp][1] = lost; }
        bool hole = false;
        if (at == 0)      // (a quarter of them each)
            for (int c = (g & 3) * 256 + tid; c < (few_whole(q) * kFewTile + p.page_size - 1) / p.page_size; c += 1024) hole |= (unsigned)p.page_table[(long)q.slot * p.max_pages + c] >= (unsigned)p.n_pages;
        hole = __syncthreads_or(hole);
        if (tid == 0) {
            uint32_t all[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++) { all[0] |= odd[i][0]; all[1] |= odd[i][1]; }
            tail_bad[g] = all[0];
            tail_gone[g] = all[1];
            tail_holes[g] = hole;
        }
        return;
    }
    // blocks of the portions, in order: 256 portions at a time, then their tiles, 256 blocks at a time
    FewBlock* blocks = reinterpret_cast<FewBlock*>(a.plan + few_blocks_at(a.pairs));
    auto scan = [&](int v, int& total) {      // what the threads before this one have; of all
        int sum = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        __syncthreads();
        if (lane == 31) sums[warp] = sum;
        __syncthreads();
        int base = 0;
        total = 0;
        for (int i = 0; i < 8; i++) {
            if (i < warp) base += sums[i];
            total += sums[i];
        }
        return base + sum - v;
    };
    if (tid < 3) carry[tid] = 0;      // blocks, tails, tiles so far
    __syncthreads();
    for (int s0 = 0; s0 < p.n_seqs; s0 += 256) {
        const int s = s0 + tid;
        const LatentPortion q = s < p.n_seqs ? latent_portion(p, a.n_tokens, s) : LatentPortion{};
        const long rows = (long)q.count * H;
        const int nb = (int)((rows + kFewRows - 1) / kFewRows), nt = few_tails(q);
        int all_b, all_t;
        const int b0 = carry[0] + scan(nb, all_b), t0 = carry[1] + scan(nt, all_t);
        const bool room = b0 + nb <= a.block_cap && t0 + nt <= a.tail_cap;      // (portions that share tokens may not have it)
        for (int b = 0; b < nb && b0 + b < a.block_cap; b++) {
            // (rows side by side hold the call's max_kv of a portion and no more: what a call says of more is not there)
            const int lead = b * kFewRows, n = (int)min((long)kFewRows, rows - lead), all = min(q.pos + (lead + n - 1) / H + 1, q.end), keys = a.rows_plan ? min(all, a.rows_plan[kPlanSeqs + p.n_seqs + 1 + s]) : all;
            blocks[b0 + b] = FewBlock{q.first * H + lead, n, lead, s, q.pos, 0, room ? (keys + kFewTile - 1) / kFewTile : 0, t0, 0, 0, 0, few_whole(q)};
        }
        __syncthreads();
        if (tid == 0) { carry[0] += all_b; carry[1] += all_t; }
        __syncthreads();
    }
    const int nb = min(carry[0], a.block_cap);
    for (int b0 = 0; b0 < nb; b0 += 256) {
        int all;
        const int b = b0 + tid, at = carry[2] + scan(b < nb ? blocks[b].tiles : 0, all);
        if (b < nb) blocks[b].tile0 = at;
        __syncthreads();
        if (tid == 0) carry[2] += all;
        __syncthreads();
    }
    const int line = carry[2], runs = min(a.pairs, (line + kFewRun - 1) / kFewRun);
    if (tid == 0) { a.plan[kFewLine] = line; a.plan[kFewBlocks] = nb; a.plan[kFewRuns] = runs; }
    for (int b = tid; b < nb; b += 256) {      // each block finds its runs, and is the first of those that begin in it
        const int x = blocks[b].tile0, n = blocks[b].tiles;
        if (n == 0) continue;
        const int first = latent_run_of(line, runs, x), last = latent_run_of(line, runs, x + n - 1);
        blocks[b].run0 = first;
        blocks[b].parts = last - first + 1;
        blocks[b].late = latent_run(line, runs, first) < x;
        for (int i = first; i <= last; i++) {
            const int at = latent_run(line, runs, i);
            if (at < x) continue;
            a.plan[kFewPairs + 2 * i] = b;
            a.plan[kFewPairs + 2 * i + 1] = at - x;
        }
    }
}

struct FewMaps { CUtensorMap q, q_rot, rows, tails; };

// Four products of the pair, O += P V: operands of consecutive K-steps 32 bytes of P's rows and 16 rows of V apart
__device__ __forceinline__ void few_mma_pv_x4(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, q, t;\n"
        ".reg .b32 r;\n"
        ".reg .b64 a, b;\n"
        "elect.sync r|q, 0xffffffff;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "setp.eq.b32 t, %4, %4;\n"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
        "add.u64 a, %1, 2;\n"
        "add.u64 b, %2, 128;\n"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, t;\n"
        "add.u64 a, a, 2;\n"
        "add.u64 b, b, 128;\n"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, t;\n"
        "add.u64 a, a, 2;\n"
        "add.u64 b, b, 128;\n"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, t;\n"
        "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void few_arrive_first(uint32_t bar) {      // at the first CTA's barrier
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(lx_cluster_at(bar, 0)) : "memory");
}

__global__ void __launch_bounds__(kFewThreads, 1) __cluster_dims__(2, 1, 1) latent_few_kernel(const __grid_constant__ FewMaps maps, const LatentFew a) {
    using namespace umma;
    extern __shared__ __align__(16) uint8_t few_smem_raw[];
    const uint32_t raw = smem_u32(few_smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* smem = few_smem_raw + (base - raw);
    FewMisc& misc = *reinterpret_cast<FewMisc*>(smem + kFewRoom);
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform(tid >> 5), rank = blockIdx.x & 1, pair = blockIdx.x >> 1;
    griddep_launch_dependents();
    if (tid == 0) {
        bar_init(smem_u32(&misc.q_full), 1); bar_init(smem_u32(&misc.q_free), 1);
        for (int i = 0; i < kFewK; i++) { bar_init(smem_u32(&misc.k_full[i]), 1); bar_init(smem_u32(&misc.k_free[i]), 1); }
        for (int i = 0; i < 4; i++) { bar_init(smem_u32(&misc.v_full[i]), 1); bar_init(smem_u32(&misc.v_free[i]), 1); }
        for (int i = 0; i < 2; i++) bar_init(smem_u32(&misc.s_full[i]), 1);
        bar_init(smem_u32(&misc.p_full), 8); bar_init(smem_u32(&misc.pv_done), 1); bar_init(smem_u32(&misc.o_free), 8);
        bar_fence_init();
        tma_prefetch_desc(&maps.q);
        tma_prefetch_desc(&maps.q_rot);
        tma_prefetch_desc(&maps.rows);
        tma_prefetch_desc(&maps.tails);
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
    const int line = a.plan[kFewLine], runs = a.plan[kFewRuns], H = a.p.heads;
    const FewBlock* blocks = reinterpret_cast<const FewBlock*>(a.plan + few_blocks_at(a.pairs));
    const int b_first = a.plan[kFewPairs + 2 * pair], t_first = a.plan[kFewPairs + 2 * pair + 1], total = pair < runs ? latent_run(line, runs, pair + 1) - latent_run(line, runs, pair) : 0;
    // every role walks the pair's run the same way: segment by segment (a block's tiles t .. t + n - 1)
    if (warp == 0) {
        // ================================================================ copies
        int left = total, b = b_first, t = t_first, it = 0, seg = 0;
        const int subs = 64 / a.box, none = a.rows_plan ? a.rows_plan[kPlanRows] : a.p.n_pages * a.p.page_size;      // (rows from there on are zeros)
        while (left > 0) {
            const FewBlock k = blocks[b];
            if (k.tiles == 0) { b++; continue; }
            const int n = min(left, k.tiles - t), slot = a.rows_plan ? 0 : a.p.slot[a.p.seqs[k.seq]], off = a.rows_plan ? a.rows_plan[kPlanSeqs + k.seq] : 0, tail = k.whole;
            const int* table = a.p.page_table + (long)slot * a.p.max_pages;
            // lane i: the row of the tile's keys from 32 i on (four of them), of the tile after the one being loaded
            auto row_of = [&](int tile) {
                if (a.rows_plan) return off + tile * kFewTile + 32 * (lane & 3);
                if (tile >= tail) return (k.tail + tile - tail) * kFewTile + 32 * (lane & 3);
                const int key = tile * kFewTile + 32 * (lane & 3), page = table[key / a.p.page_size];
                return (unsigned)page < (unsigned)a.p.n_pages ? page * a.p.page_size + key % a.p.page_size : none;
            };
            int row = row_of(t);
            if (lane == 0) {
                bar_wait(smem_u32(&misc.q_free), (seg & 1) ^ 1);
                if (rank == 0) bar_expect_tx(smem_u32(&misc.q_full), 2 * kFewK * kFewBox);
                const uint32_t bar = lx_cluster_at(smem_u32(&misc.q_full), 0);
                for (int c = 0; c < 8; c++) lx_load_pair(base + c * kFewBox, &maps.q, bar, c * 64, k.row0 + 64 * rank);
                lx_load_pair(base + 8 * kFewBox, &maps.q_rot, bar, 0, k.row0 + 64 * rank);
            }
            __syncwarp();
            auto keys = [&](int tile, int r, int i) {      // the pair's i-th tile so far
                const CUtensorMap* m = !a.rows_plan && tile >= tail ? &maps.tails : &maps.rows;
                const int r0 = __shfl_sync(0xffffffffu, r, 2 * rank), r1 = __shfl_sync(0xffffffffu, r, 2 * rank + 1);
                if (lane == 0)
                    for (int c = 0; c < kFewK; c++) {
                        bar_wait(smem_u32(&misc.k_free[c]), (i & 1) ^ 1);
                        const uint32_t dst = base + kFewOffK + c * kFewBox, bar = lx_cluster_at(smem_u32(&misc.k_full[c]), 0);
                        if (rank == 0) bar_expect_tx(smem_u32(&misc.k_full[c]), 2 * kFewBox);
                        lx_load_pair(dst, m, bar, c * 64, r0);
                        if (subs == 2) lx_load_pair(dst + kFewBox / 2, m, bar, c * 64, r1);
                    }
                __syncwarp();
            };
            auto values = [&](int tile, int r, int i) {
                const CUtensorMap* m = !a.rows_plan && tile >= tail ? &maps.tails : &maps.rows;
                const int r0 = __shfl_sync(0xffffffffu, r, 0), r1 = __shfl_sync(0xffffffffu, r, 1), r2 = __shfl_sync(0xffffffffu, r, 2), r3 = __shfl_sync(0xffffffffu, r, 3);
                if (lane == 0)
                    for (int g = 0; g < 4; g++) {      // [half of the keys][256 columns]: this CTA's 128 of them
                        bar_wait(smem_u32(&misc.v_free[g]), (i & 1) ^ 1);
                        const uint32_t bar = lx_cluster_at(smem_u32(&misc.v_full[g]), 0);
                        if (rank == 0) bar_expect_tx(smem_u32(&misc.v_full[g]), 4 * kFewBox);
                        for (int x = 0; x < 2; x++) {
                            const uint32_t dst = base + kFewOffV + (2 * g + x) * kFewBox;
                            const int c = (g & 1) * 256 + rank * 128 + x * 64;
                            lx_load_pair(dst, m, bar, c, g < 2 ? r0 : r2);
                            if (subs == 2) lx_load_pair(dst + kFewBox / 2, m, bar, c, g < 2 ? r1 : r3);
                        }
                    }
                __syncwarp();
            };
            // in the order in which the products give room: keys of a tile ahead of the values of the one before it
            keys(t, row, it);
            for (int j = 0; j < n; j++) {
                const int next = j + 1 < n ? row_of(t + j + 1) : 0;
                if (j + 1 < n) keys(t + j + 1, next, it + j + 1);
                values(t + j, row, it + j);
                row = next;
            }
            it += n;
            left -= n;
            seg++;
            b++;
            t = 0;
        }
    } else if (warp == 1 && rank == 0) {
        // ================================================================ products (converged warp)
        constexpr uint32_t idesc_qk = instr_desc(1, 1, 1, 0, 0, 128, 128), idesc_pv = instr_desc(1, 1, 1, 0, 1, 128, 256);      // V [key][column]: B MN-major
        int left = total, b = b_first, t = t_first, it = 0, seg = 0;
        while (left > 0) {
            const int tiles = blocks[b].tiles, n = min(left, tiles - t);
            if (tiles == 0) { b++; continue; }
            auto scores = [&](int i, bool last) {
#pragma unroll 1
                for (int c = 0; c < kFewK; c++) {
                    bar_wait(smem_u32(&misc.k_full[c]), i & 1);
                    tc_fence_after();
                    lx_mma_pair_x4(tmem + 256 + (i & 1) * 64, smem_desc(base + c * kFewBox, 16, 1024, kLayoutSw128), smem_desc(base + kFewOffK + c * kFewBox, 16, 1024, kLayoutSw128), idesc_qk, c > 0,
                                   smem_u32(&misc.k_free[c]), c == kFewK - 1 ? smem_u32(&misc.s_full[i & 1]) : 0);
                }
                if (last) lx_commit_pair(smem_u32(&misc.q_free));
            };
            bar_wait(smem_u32(&misc.q_full), seg & 1);
            scores(it, n == 1);
            for (int j = 0; j < n; j++) {
                if (j + 1 < n) scores(it + j + 1, j + 2 == n);
                if (j == 0) bar_wait(smem_u32(&misc.o_free), (seg & 1) ^ 1);      // (the results of the segment before are read)
                bar_wait(smem_u32(&misc.p_full), (it + j) & 1);
                tc_fence_after();
#pragma unroll 1
                for (int g = 0; g < 4; g++) {
                    bar_wait(smem_u32(&misc.v_full[g]), (it + j) & 1);
                    tc_fence_after();
                    few_mma_pv_x4(tmem + (g & 1) * 128, smem_desc(base + kFewOffP + (g >> 1) * kFewBox, 16, 1024, kLayoutSw128), smem_desc(base + kFewOffV + 2 * g * kFewBox, kFewBox, 1024, kLayoutSw128), idesc_pv,
                                  j > 0 || g > 1);
                    lx_commit_pair(smem_u32(&misc.v_free[g]));
                }
                lx_commit_pair(smem_u32(&misc.pv_done));
            }
            it += n;
            left -= n;
            seg++;
            b++;
            t = 0;
        }
    } else if (warp >= 2) {
        // ================================================================ soft-max
        const int sp = warp & 3, half = sp >> 1, r = 32 * (sp & 1) + lane;      // TMEM lane 32 sp + lane: the row r and the tile's keys (or O's columns) of this half
        const uint32_t tl = tmem + ((uint32_t)(32 * sp) << 16);
        const float c = a.scale_log2;
        const int room = latent_room(a.p);
        const bool odd = a.rows_plan && a.rows_plan[kPlanOdd] != 0;      // (rows side by side are copies, all of them; other tiles ahead of the tails are as the cache holds them)
        int left = total, b = b_first, t = t_first, it = 0, seg = 0;
        while (left > 0) {
            const FewBlock k = blocks[b];
            if (k.tiles == 0) { b++; continue; }
            const int n = min(left, k.tiles - t), in = 64 * rank + r, tail = k.whole;
            const bool valid = in < k.rows;
            const int p = valid ? min(k.pos0 + (k.lead + in) / H, room - 1) : -1;      // the last key that the row sees
            const int* table = a.p.page_table + (a.rows_plan ? 0 : (long)a.p.slot[a.p.seqs[k.seq]] * a.p.max_pages);
            float m_ref = -INFINITY, l = 0.f;
            bool lost = false, holes = false;      // keys of this half were not there; there may be such
            if (!a.rows_plan && t < tail) {
                const uint4 h = a.holes[k.tail];
                holes = h.x | h.y | h.z | h.w;
            }
            for (int j = 0; j < n; j++) {
                const int i = it + j, k0 = (t + j) * kFewTile + 64 * half;
                uint2 gone = make_uint2(0, 0);
                if (t + j >= tail || a.rows_plan) {
                    if (t + j >= tail || odd) gone = *reinterpret_cast<const uint2*>(a.gone + (a.rows_plan ? a.rows_plan[kPlanSeqs + k.seq] + k0 : (k.tail + t + j - tail) * kFewTile + 64 * half) / 32);
                } else if (holes) {
                    gone.x = (unsigned)table[k0 / a.p.page_size] < (unsigned)a.p.n_pages ? 0 : 0xffffffffu;
                    gone.y = a.box == 64 ? gone.x : (unsigned)table[(k0 + 32) / a.p.page_size] < (unsigned)a.p.n_pages ? 0 : 0xffffffffu;
                }
                bar_wait(smem_u32(&misc.s_full[i & 1]), (i >> 1) & 1);
                tc_fence_after();
                float s[64];
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    uint32_t v[32];
                    tmem_ld32(tl + 256 + (i & 1) * 64 + 32 * q, v);
#pragma unroll
                    for (int x = 0; x < 32; x++) s[32 * q + x] = __uint_as_float(v[x]);
                }
                tmem_wait_ld();
                // (the loads above are in registers only now)
#pragma unroll
                for (int x = 0; x < 64; x++) asm volatile("" : "+f"(s[x]));
                if (odd || t + j >= tail) {
                    const uint2 w = *reinterpret_cast<const uint2*>(a.bad + (a.rows_plan ? a.rows_plan[kPlanSeqs + k.seq] + k0 : (k.tail + t + j - tail) * kFewTile + 64 * half) / 32);
                    if (w.x | w.y) {
#pragma unroll
                        for (int x = 0; x < 64; x++)
                            if ((x < 32 ? w.x : w.y) >> (x & 31) & 1) s[x] = __int_as_float(0x7fffffff);
                    }
                }
                if (gone.x | gone.y) {
                    lost = true;
#pragma unroll
                    for (int x = 0; x < 64; x++)
                        if ((x < 32 ? gone.x : gone.y) >> (x & 31) & 1) s[x] = -INFINITY;
                }
                if (t + j >= tail) {      // (a tile that not all rows see whole, or one of the portion's last)
                    const int i1 = p - k0;
#pragma unroll
                    for (int x = 0; x < 64; x++)
                        if (x > i1) s[x] = -INFINITY;
                }
                float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int x = 4; x < 64; x += 4)
#pragma unroll
                    for (int q = 0; q < 4; q++) mx[q] = fmaxf(mx[q], s[x + q]);
                const float mine = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c;
                misc.top[i & 1][half][r] = mine;
                asm volatile("barrier.cta.sync 1, 128;" ::: "memory");
                const float m_new = fmaxf(mine, misc.top[i & 1][half ^ 1][r]);
                const bool raise = m_new > m_ref + 8.f || (m_ref == -INFINITY && m_new > -INFINITY);
                const float m_old = m_ref;
                if (raise) m_ref = m_new;
                const float u = m_ref == -INFINITY ? 0.f : m_ref;
                const f32x2 c2 = pack2(c, c), o2 = pack2(-u, -u);
                f32x2 sum[2] = {0, 0};
                uint32_t pk[32];
#pragma unroll
                for (int x = 0; x < 32; x++) {
                    float e0, e1;
                    unpack2(fma2(pack2(s[2 * x], s[2 * x + 1]), c2, o2), e0, e1);
                    e0 = latent_exp2(e0);
                    e1 = latent_exp2(e1);
                    pk[x] = latent_pack(e0, e1);
                    sum[x & 1] = add2(sum[x & 1], pack2(e0, e1));
                }
                if (i > 0) {      // P and O of the tile before are done with
                    bar_wait(smem_u32(&misc.pv_done), (i - 1) & 1);
                    tc_fence_after();
                }
                if (__any_sync(0xffffffffu, raise) && j > 0) {
                    const float alpha = raise ? latent_exp2(m_old - m_ref) : 1.f;
                    l *= alpha;
#pragma unroll 1
                    for (int q = 0; q < 8; q++) {
                        uint32_t v[32];
                        tmem_ld32(tl + 32 * q, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int x = 0; x < 32; x++) v[x] = __float_as_uint(__uint_as_float(v[x]) * alpha);
                        tmem_st32(tl + 32 * q, v);
                    }
                    tmem_wait_st();
                }
                uint8_t* to = smem + kFewOffP + half * kFewBox + r * 128;
#pragma unroll
                for (int x = 0; x < 8; x++) *reinterpret_cast<uint4*>(to + ((x ^ (r & 7)) << 4)) = make_uint4(pk[4 * x], pk[4 * x + 1], pk[4 * x + 2], pk[4 * x + 3]);
                fence_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) few_arrive_first(smem_u32(&misc.p_full));
                float a0, a1, a2, a3;
                unpack2(sum[0], a0, a1);
                unpack2(sum[1], a2, a3);
                l += (a0 + a1) + (a2 + a3);
            }
            it += n;
            // ---- the segment's result
            bar_wait(smem_u32(&misc.pv_done), (it - 1) & 1);
            tc_fence_after();
            asm volatile("barrier.cta.sync 1, 128;" ::: "memory");      // (the maxima are read)
            l = latent_sum(l, lost);
            misc.top[0][half][r] = l;
            asm volatile("barrier.cta.sync 1, 128;" ::: "memory");
            const float other = misc.top[0][half ^ 1][r];
            l = latent_sum(l + other, __float_as_uint(l) == kNoKeys || __float_as_uint(other) == kNoKeys);
            asm volatile("barrier.cta.sync 1, 128;" ::: "memory");
            const bool whole = n == k.tiles;
            const long row = (long)k.row0 + in, part = 2L * pair + (seg > 0);
            const float inv = latent_inverse(l);
            if (!whole && valid && half == 0) *reinterpret_cast<float2*>(a.ml_part + (part * kFewRows + in) * 2) = make_float2(m_ref, l);
#pragma unroll 1
            for (int q = 0; q < 8; q++) {      // 128 columns from 128 half on of each 256
                uint32_t v[32];
                tmem_ld32(tl + 32 * q, v);
                tmem_wait_ld();
                if (!valid) continue;
                const int col = (q >> 2) * 256 + 128 * half + (q & 3) * 32;
                if (whole) {
                    uint32_t o[16];
#pragma unroll
                    for (int x = 0; x < 16; x++) o[x] = latent_pack(__uint_as_float(v[2 * x]) * inv, __uint_as_float(v[2 * x + 1]) * inv);
                    __nv_bfloat16* to = a.sums + row * kLatent + col;
                    latent_store32(to, o);
                    latent_store32(to + 16, o + 8);
                } else {
                    float* to = a.o_part + (part * kFewRows + in) * kLatent + col;
#pragma unroll
                    for (int x = 0; x < 4; x++) latent_store32(to + 8 * x, v + 8 * x);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) few_arrive_first(smem_u32(&misc.o_free));
            left -= n;
            seg++;
            b++;
            t = 0;
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

// joins the parts of blocks that were cut: a warp a row, grid (blocks, 16)
__global__ void __launch_bounds__(256) latent_few_merge_kernel(const LatentFew a) {
    griddep_launch_dependents();
    griddep_wait();
    const int lane = threadIdx.x & 31, in = blockIdx.y * 8 + (threadIdx.x >> 5);
    if ((int)blockIdx.x >= a.plan[kFewBlocks]) return;
    const FewBlock k = reinterpret_cast<const FewBlock*>(a.plan + few_blocks_at(a.pairs))[blockIdx.x];
    if (in >= k.rows || k.tiles == 0 || k.parts == 1) return;
    const int parts = k.parts;
    auto at = [&](int i) { return (2L * (k.run0 + i) + (i == 0 ? k.late : 0)) * kFewRows + in; };
    float m = -INFINITY, l = 0.f, o[16];
    bool nan = false, gone = false;
#pragma unroll
    for (int x = 0; x < 16; x++) o[x] = 0.f;
    for (int i = lane; i < parts; i += 32) m = fmaxf(m, a.ml_part[at(i) * 2]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
#pragma unroll 4
    for (int i = 0; i < parts; i++) {
        const float2 ml = *reinterpret_cast<const float2*>(a.ml_part + at(i) * 2);
        float4 v[4];
#pragma unroll
        for (int x = 0; x < 4; x++) v[x] = *reinterpret_cast<const float4*>(a.o_part + at(i) * kLatent + x * 128 + lane * 4);
        nan |= ml.y != ml.y;
        gone |= __float_as_uint(ml.y) == kNoKeys;
        const float w = ml.x == -INFINITY ? 0.f : latent_exp2(ml.x - m);      // (0: what is not finite in the part's sum still makes the row NaN)
        l = fmaf(ml.y, w, l);
#pragma unroll
        for (int x = 0; x < 4; x++) { o[4 * x] = fmaf(v[x].x, w, o[4 * x]); o[4 * x + 1] = fmaf(v[x].y, w, o[4 * x + 1]); o[4 * x + 2] = fmaf(v[x].z, w, o[4 * x + 2]); o[4 * x + 3] = fmaf(v[x].w, w, o[4 * x + 3]); }
    }
    const float inv = nan ? __int_as_float(0x7fffffff) : latent_inverse(latent_sum(l, gone));
    __nv_bfloat16* to = a.sums + ((long)k.row0 + in) * kLatent;
#pragma unroll
    for (int x = 0; x < 4; x++) *reinterpret_cast<uint2*>(to + x * 128 + lane * 4) = make_uint2(latent_pack(o[4 * x] * inv, o[4 * x + 1] * inv), latent_pack(o[4 * x + 2] * inv, o[4 * x + 3] * inv));
}

}  // namespace ktb
