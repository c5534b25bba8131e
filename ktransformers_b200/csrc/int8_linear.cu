// Linear with 8-bit integers: a scale per token for the activations, a scale per output channel for the weights.
//     s[t] = max_k |x[t][k]| * (1 / 127) (fp32),  c[t][k] = rint(x[t][k] / s[t])                     (IEEE quotient; 0 where the row is zero)
//     y[t][n] = cast(float(sum_k c[t][k] w[n][k]) * (s[t] w_scale[n]) + bias[n])                 (the sum in 32-bit integers, exact)
// A row of x with an infinity or NaN has no scale: its results are NaN.
//
// int8_quant_kernel makes codes and scales, a row per CTA.  Then one of two products on tcgen05.mma.kind::i8, whose 32-bit sums stay in tensor memory over all of K and are exact in
// any order (so that splits of K join without rounding):
//   int8_rows_kernel   weight rows on the MMA's 128 rows, 16 to 128 tokens on its columns: a decode step reads the weights once.  K is split over the CTAs of a cluster, which add their
//                      parts through distributed shared memory: no workspace to clear, no second launch.  Weight boxes are under way before the codes are there (the launch is
//                      a programmatic dependent of the quantiser's, which lets it start once all work ahead of the call is complete).
//   int8_gemm_kernel   prompts: 256 tokens x up to 256 outputs a tile of two CTAs, persistent, two accumulators in tensor memory
#include <cuda.h>

#include <algorithm>
#include <climits>

#include "common.cuh"
#include "umma.cuh"

namespace ktb {
using namespace umma;

// ------------------------------------------------------------------------------------------------ codes
// A row per CTA: the largest magnitude, then the codes; codes behind column K (up to Kp) are zeros.  VEC: rows of whole 16-byte vectors, of which a thread keeps kI8Keep in registers between
// the two (what does not fit is read again, from L2).  Bound by the bytes of x and of the codes, and by little: nine instructions a value.
//   - magnitudes are compared as their bits (two 16-bit ones at a time); infinities and NaN are the largest of all
//   - a code is rint of the fp32 quotient x / s.  x times 1 / s is within 2e-5 of that, so its nearest integer (an addition of 1.5 2^23) is the code unless it stands so close to the middle
//     of two; a vector with such a value, one in some thousand, is divided.  (Divided throughout 4000 rows of 18432 took 130 us.)
constexpr int kI8Keep = 6;
constexpr float kI8Magic = 12582912.f;      // 1.5 2^23: the low byte of magic + k is k's
template <int TYPE> __device__ __forceinline__ void i8_unpack(uint4 w, float (&v)[TYPE == KTB200_TYPE_F32 ? 4 : 8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (TYPE == KTB200_TYPE_F32) v[i] = __uint_as_float(u[i]);
        else if constexpr (TYPE == KTB200_TYPE_BF16) { v[2 * i] = __uint_as_float(u[i] << 16); v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
        else { v[2 * i] = fp16_bits_to_f32((uint16_t)u[i]); v[2 * i + 1] = fp16_bits_to_f32((uint16_t)(u[i] >> 16)); }
    }
}
__device__ __forceinline__ uint32_t i8_code(float x, float s) { return (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(x, s)), -127.f), 127.f) & 0xffu; }
// the magnitude of a value of the type, from its bits
template <int TYPE> __device__ __forceinline__ float i8_magnitude(uint32_t bits) {
    return TYPE == KTB200_TYPE_F32 ? __uint_as_float(bits) : TYPE == KTB200_TYPE_BF16 ? __uint_as_float(bits << 16) : fp16_bits_to_f32((uint16_t)bits);
}
template <int TYPE> __device__ __forceinline__ uint32_t i8_bits(const uint8_t* row, int k) {
    if constexpr (TYPE == KTB200_TYPE_F32) return reinterpret_cast<const uint32_t*>(row)[k] & 0x7fffffffu;
    else return reinterpret_cast<const uint16_t*>(row)[k] & 0x7fffu;
}

template <int TYPE, bool VEC> __global__ void __launch_bounds__(512) int8_quant_kernel(const void* x, long x_stride, int K, int Kp, int8_t* codes, float* scales) {
    constexpr int E = TYPE == KTB200_TYPE_F32 ? 4 : 8, ESZ = 16 / E;
    constexpr uint32_t kInf = TYPE == KTB200_TYPE_F32 ? 0x7f800000u : TYPE == KTB200_TYPE_BF16 ? 0x7f80u : 0x7c00u;
    __shared__ uint32_t red[16];
    const long t = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    griddep_wait();
    griddep_launch_dependents();      // (behind the wait: the rows kernel asks for weights as soon as it starts, and what is ahead of this kernel in the stream may have made them)
    uint32_t top = 0;      // 16-bit types: of the even and of the odd values
    uint4 keep[VEC ? kI8Keep : 1];
    const uint8_t* row = reinterpret_cast<const uint8_t*>(x) + t * x_stride * ESZ;
    auto largest = [&](uint4 w) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) top = TYPE == KTB200_TYPE_F32 ? max(top, u[i] & 0x7fffffffu) : __vmaxu2(top, u[i] & 0x7fff7fffu);
    };
    if constexpr (VEC) {
        const int n = K / E;
#pragma unroll
        for (int i = 0; i < kI8Keep; i++) {
            const int at = threadIdx.x + i * blockDim.x;
            keep[i] = at < n ? *reinterpret_cast<const uint4*>(row + 16 * (long)at) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kI8Keep; i++) largest(keep[i]);
        for (int at = threadIdx.x + kI8Keep * blockDim.x; at < n; at += blockDim.x) largest(*reinterpret_cast<const uint4*>(row + 16 * (long)at));
        if constexpr (TYPE != KTB200_TYPE_F32) top = max(top & 0xffffu, top >> 16);
    } else {
        for (int k = threadIdx.x; k < K; k += blockDim.x) top = max(top, i8_bits<TYPE>(row, k));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) red[warp] = top;
    __syncthreads();
    top = red[0];
    for (int w = 1; w < nw; w++) top = max(top, red[w]);
    const float s = top >= kInf ? NAN : i8_magnitude<TYPE>(top) * (1.0f / 127.0f);      // (by the rounded inverse, as tensor arithmetic on the GPU divides by a number: the codes are the same as there)
    const bool some = s > 0.f;
    if (threadIdx.x == 0) scales[t] = s;
    int8_t* out = codes + t * Kp;
    if constexpr (VEC) {
        const float inv = s > 1e-37f ? __fdiv_rn(1.0f, s) : 0.f;      // (0: scales whose inverse fp32 does not hold; their rows are divided)
        auto store = [&](int at, uint4 w) {
            float v[E], far = inv > 0.f ? 0.f : 1.f;
            i8_unpack<TYPE>(w, v);
            uint32_t c[E / 4] = {}, r[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float m = fmaf(v[e], inv, kI8Magic);
                far = fmaxf(far, fabsf(fmaf(v[e], inv, kI8Magic - m)));
                r[e] = __float_as_uint(m);
            }
#pragma unroll
            for (int i = 0; i < E / 4; i++) c[i] = __byte_perm(__byte_perm(r[4 * i], r[4 * i + 1], 0x0040), __byte_perm(r[4 * i + 2], r[4 * i + 3], 0x0040), 0x5410);
            if (far > 0.4999f) {
#pragma unroll
                for (int i = 0; i < E / 4; i++) c[i] = 0;
                if (some) {
#pragma unroll
                    for (int e = 0; e < E; e++) c[e / 4] |= i8_code(v[e], s) << (8 * (e & 3));
                }
            }
            if constexpr (E == 4) *reinterpret_cast<uint32_t*>(out + 4 * (long)at) = c[0];
            else *reinterpret_cast<uint2*>(out + 8 * (long)at) = make_uint2(c[0], c[1]);
        };
        const int n = K / E;
#pragma unroll
        for (int i = 0; i < kI8Keep; i++) {
            const int at = threadIdx.x + i * blockDim.x;
            if (at < n) store(at, keep[i]);
        }
        for (int at = threadIdx.x + kI8Keep * blockDim.x; at < n; at += blockDim.x) store(at, *reinterpret_cast<const uint4*>(row + 16 * (long)at));
        for (int k = K + threadIdx.x; k < Kp; k += blockDim.x) out[k] = 0;
    } else {
        for (int k = threadIdx.x; k < Kp; k += blockDim.x) out[k] = k < K && some ? (int8_t)i8_code(load_hidden(row, k, TYPE), s) : (int8_t)0;
    }
}

struct Int8Out {
    const float *xs, *ws, *bias;      // scale of each token, of each output, and the outputs' biases or null
    void* y;
    long y_stride;
    const int* bsz;
    int type, T, N, nkb;
};
__device__ __forceinline__ float i8_result(int acc, float xs, float ws, float bias) { return __fadd_rn(__fmul_rn((float)acc, __fmul_rn(xs, ws)), bias); }

// ------------------------------------------------------------------------------------------------ few tokens
// grid (row tiles of 128, K splits = the cluster, token tiles of NT); 192 threads: warp 0 copies, warp 1 products, warps 2-5 results.  A stage of the ring is 128 bytes of K: a box of
// 128 weight rows and one of NT tokens.
constexpr int kI8RowsThreads = 192, kI8MaxSplits = 8;
template <int NT> constexpr int i8_rows_stage() { return 128 * 128 + NT * 128; }
template <int NT> constexpr int i8_rows_stages() { return NT == 16 ? 6 : NT == 32 ? 5 : NT == 64 ? 4 : 3; }      // about 100 KB: two CTAs an SM
struct Int8RowsMisc {
    unsigned long long full[6], free[6], done;
    uint32_t tmem_base;
};
template <int NT> constexpr int i8_rows_smem() { return i8_rows_stages<NT>() * i8_rows_stage<NT>() + (int)sizeof(Int8RowsMisc) + 1024; }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ int cluster_load(uint32_t addr, uint32_t rank) {      // a word of another CTA's shared memory
    uint32_t at;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at));      // (ordered by the cluster's barriers)
    return v;
}

template <int NT> __global__ void __launch_bounds__(kI8RowsThreads, 2) int8_rows_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Int8Out o, int per) {
    constexpr int STAGE = i8_rows_stage<NT>(), STAGES = i8_rows_stages<NT>(), COLS = NT < 32 ? 32 : NT;
    extern __shared__ __align__(16) uint8_t i8_smem_raw[];
    const uint32_t raw = smem_u32(i8_smem_raw), base = (raw + 1023u) & ~1023u;
    Int8RowsMisc& misc = *reinterpret_cast<Int8RowsMisc*>(i8_smem_raw + (base - raw) + STAGES * STAGE);
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform(tid >> 5), n0 = blockIdx.x * 128, t0 = blockIdx.z * NT, kb0 = blockIdx.y * per, nk = min(per, o.nkb - kb0);
    griddep_launch_dependents();
    if (tid == 0) {
        for (int i = 0; i < STAGES; i++) { bar_init(smem_u32(&misc.full[i]), 1); bar_init(smem_u32(&misc.free[i]), 1); }
        bar_init(smem_u32(&misc.done), 1);
        bar_fence_init();
        tma_prefetch_desc(&wmap);
        tma_prefetch_desc(&xmap);
    }
    if (warp == 1) tmem_alloc(smem_u32(&misc.tmem_base), COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = uniform(misc.tmem_base);
    if (warp == 0) {
        if (lane == 0) {
            // the ring's first weights do not wait for the codes (what was ahead of the quantiser is complete: it lets this kernel start behind its own wait)
            for (int i = 0; i < nk && i < STAGES; i++) {
                const uint32_t bar = smem_u32(&misc.full[i]);
                bar_expect_tx(bar, STAGE);
                tma_load_2d(base + i * STAGE, &wmap, bar, (kb0 + i) * 128, n0);
            }
            griddep_wait();
            for (int i = 0; i < nk && i < STAGES; i++) tma_load_2d(base + i * STAGE + 128 * 128, &xmap, smem_u32(&misc.full[i]), (kb0 + i) * 128, t0);
            for (int i = STAGES; i < nk; i++) {
                const int s = i % STAGES;
                const uint32_t bar = smem_u32(&misc.full[s]);
                bar_wait(smem_u32(&misc.free[s]), ((i / STAGES) & 1) ^ 1);
                bar_expect_tx(bar, STAGE);
                tma_load_2d(base + s * STAGE, &wmap, bar, (kb0 + i) * 128, n0);
                tma_load_2d(base + s * STAGE + 128 * 128, &xmap, bar, (kb0 + i) * 128, t0);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        constexpr uint32_t idesc = instr_desc(2, 1, 1, 0, 0, 128, NT);      // s32 += s8 . s8, K-major both
        for (int i = 0; i < nk; i++) {
            const int s = i % STAGES;
            bar_wait(smem_u32(&misc.full[s]), (i / STAGES) & 1);
            tc_fence_after();
            mma_i8_x4(tmem, smem_desc(base + s * STAGE, 16, 1024, kLayoutSw128), smem_desc(base + s * STAGE + 128 * 128, 16, 1024, kLayoutSw128), idesc, i > 0, smem_u32(&misc.free[s]),
                      i + 1 == nk ? smem_u32(&misc.done) : 0);
        }
    }
    const int splits = gridDim.y, sp = warp & 3, r = 32 * sp + lane, n = n0 + r, live = min(o.T - t0, NT);
    if (warp >= 2) {
        griddep_wait();      // (the tokens' scales)
        bar_wait(smem_u32(&misc.done), 0);
        tc_fence_after();
        const int mine = o.bsz ? min(live, *o.bsz - t0) : live;
        const float ws = n < o.N ? o.ws[n] : 0.f, bias = n < o.N && o.bias ? o.bias[n] : 0.f;
        int* part = reinterpret_cast<int*>(i8_smem_raw + (base - raw));      // [NT][128] over the ring, which the products are done with
#pragma unroll 1
        for (int c = 0; c < NT; c += 16) {
            if (c >= live) break;
            uint32_t v[16];
            tmem_ld16(tmem + ((uint32_t)(32 * sp) << 16) + c, v);
            tmem_wait_ld();
            if (splits > 1) {
#pragma unroll
                for (int i = 0; i < 16; i++) part[(c + i) * 128 + r] = (int)v[i];
            } else if (n < o.N) {
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (c + i < mine) store_hidden(o.y, (long)(t0 + c + i) * o.y_stride + n, o.type, i8_result((int)v[i], __ldg(o.xs + t0 + c + i), ws, bias));
            }
        }
        tc_fence_before();
    }
    if (splits > 1) {      // rank k of the cluster adds up the tokens k, k + splits, ..
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (warp >= 2) {
            const int mine = o.bsz ? min(live, *o.bsz - t0) : live;
            const float ws = n < o.N ? o.ws[n] : 0.f, bias = n < o.N && o.bias ? o.bias[n] : 0.f;
            // four tokens at a time, so that the loads from all CTAs of the cluster are on their way together
            for (int t0c = blockIdx.y; t0c < mine; t0c += 4 * splits) {
                int v[4][kI8MaxSplits];
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int k = 0; k < kI8MaxSplits; k++) v[i][k] = k < splits && t0c + i * splits < mine ? cluster_load(base + ((t0c + i * splits) * 128 + r) * 4, k) : 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = t0c + i * splits;
                    int acc = 0;
#pragma unroll
                    for (int k = 0; k < kI8MaxSplits; k++) acc += v[i][k];
                    if (t < mine && n < o.N) store_hidden(o.y, (long)(t0 + t) * o.y_stride + n, o.type, i8_result(acc, __ldg(o.xs + t0 + t), ws, bias));
                }
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
        tmem_dealloc(tmem, COLS);
    }
}

// ------------------------------------------------------------------------------------------------ many tokens
// Persistent pairs of CTAs (cta_group::2): a pair's tile is 256 tokens x bn outputs, each CTA has 128 of the tokens and brings half of the outputs' weight rows, which both tensor
// cores read: a K block of 128 costs a CTA 16 KB + 64 bn bytes of shared memory each way where one CTA alone would need 16 KB + 128 bn (single CTAs with 256 columns were bound by
// that: 735 cycles a block against 524 of the products).  bn is any multiple of 32: the one whose rounds of tiles take least.
//     warp 0 TMA ring (192 KB) of its own half, whose bytes are counted by the first CTA's barriers; warp 1 of the first CTA the pair's products; warps 4-19 results (a thread one token,
//     every fourth run of 16 columns).  Two accumulators of bn columns.
// Tiles run token tile fastest inside groups of kI8Group, so that the CTAs of a wave share the weight rows and the tokens through L2.
constexpr int kI8GemmThreads = 640, kI8Group = 8, kI8Ring = 192 * 1024, kI8Turn = 16 * 33;
struct Int8GemmMisc {
    unsigned long long full[8], free[8], d_full[2], d_free[2];
    uint32_t tmem_base;
};
constexpr int kI8GemmSmem = kI8Ring + (int)sizeof(Int8GemmMisc) + 1024, kI8GemmSmemTurn = kI8GemmSmem + 16 * kI8Turn * 4;
static_assert(kI8GemmSmemTurn <= 232448, "shared memory budget");
__host__ __device__ constexpr int i8_gemm_stage(int bn) { return 128 * 128 + bn / 2 * 128; }
__host__ __device__ constexpr int i8_gemm_stages(int bn) { return kI8Ring / i8_gemm_stage(bn) < 8 ? kI8Ring / i8_gemm_stage(bn) : 8; }

__device__ __forceinline__ uint32_t cluster_at(uint32_t addr, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
    return at;
}
// a box into this CTA's shared memory, counted by a barrier of either CTA of the pair
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* m, uint32_t bar, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(m), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
// Four products of the pair on consecutive K-steps of 32 bytes, and the barriers (of both CTAs) that complete when all so far have (0: not asked for); called by a converged warp
__device__ __forceinline__ void mma_i8_pair_x4(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate, uint32_t bar0, uint32_t bar1) {
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
        "@q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n"
        "add.u64 a, %1, 2;\n"
        "add.u64 b, %2, 2;\n"
        "@q tcgen05.mma.cta_group::2.kind::i8 [%0], a, b, %3, t;\n"
        "add.u64 a, a, 2;\n"
        "add.u64 b, b, 2;\n"
        "@q tcgen05.mma.cta_group::2.kind::i8 [%0], a, b, %3, t;\n"
        "add.u64 a, a, 2;\n"
        "add.u64 b, b, 2;\n"
        "@q tcgen05.mma.cta_group::2.kind::i8 [%0], a, b, %3, t;\n"
        "@c tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%5], both;\n"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%6], both;\n"
        "}\n" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(bar0), "r"(bar1) : "memory");
}

// TURN: rows of y that do not begin at 32 bytes.  A thread's columns of its token would be scattered values; the warp turns 16 columns of its 32 tokens around in shared memory, and
// 16 threads write 16 columns of one row
template <bool TURN> __global__ void __launch_bounds__(kI8GemmThreads, 1) __cluster_dims__(2, 1, 1)
    int8_gemm_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap, const Int8Out o, int bn, int mt, int nt) {
    extern __shared__ __align__(16) uint8_t i8_smem_raw[];
    const uint32_t raw = smem_u32(i8_smem_raw), base = (raw + 1023u) & ~1023u;
    Int8GemmMisc& misc = *reinterpret_cast<Int8GemmMisc*>(i8_smem_raw + (base - raw) + kI8Ring);
    const int tid = threadIdx.x, lane = tid & 31, warp = uniform(tid >> 5), rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const int stage = i8_gemm_stage(bn), stages = i8_gemm_stages(bn), tiles = mt * nt;
    griddep_launch_dependents();
    if (tid == 0) {
        for (int s = 0; s < 8; s++) { bar_init(smem_u32(&misc.full[s]), 1); bar_init(smem_u32(&misc.free[s]), 1); }
        for (int b = 0; b < 2; b++) { bar_init(smem_u32(&misc.d_full[b]), 1); bar_init(smem_u32(&misc.d_free[b]), 32); }
        bar_fence_init();
        tma_prefetch_desc(&xmap);
        tma_prefetch_desc(&wmap);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&misc.tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();      // (the pair's barriers and tensor memory are there)
    cluster_wait();
    tc_fence_after();
    const uint32_t tmem = uniform(misc.tmem_base);
    auto place = [&](int tile, int& m0, int& n0) {
        const int per = kI8Group * nt, g = tile / per, r = tile - g * per, gm = min(kI8Group, mt - g * kI8Group);
        n0 = (r / gm) * bn;
        m0 = (g * kI8Group + r % gm) * 256 + rank * 128;
    };
    griddep_wait();
    if (warp == 0) {
        if (lane == 0) {
            int s = 0, ph = 1;
            for (int tile = pair; tile < tiles; tile += pairs) {
                int m0, n0;
                place(tile, m0, n0);
                for (int kb = 0; kb < o.nkb; kb++) {
                    bar_wait(smem_u32(&misc.free[s]), ph);
                    const uint32_t dst = base + s * stage, bar = cluster_at(smem_u32(&misc.full[s]), 0);
                    if (rank == 0) bar_expect_tx(smem_u32(&misc.full[s]), 2 * stage);
                    tma_load_pair(dst, &xmap, bar, kb * 128, m0);
                    tma_load_pair(dst + 128 * 128, &wmap, bar, kb * 128, n0 + rank * (bn / 2));
                    if (++s == stages) { s = 0; ph ^= 1; }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1 && rank == 0) {
        const uint32_t idesc = instr_desc(2, 1, 1, 0, 0, 256, 0) | ((uint32_t)(bn >> 3) << 17);
        int s = 0, ph = 0, it = 0;
        for (int tile = pair; tile < tiles; tile += pairs, it++) {
            const int buf = it & 1;
            bar_wait(smem_u32(&misc.d_free[buf]), ((it >> 1) & 1) ^ 1);
            tc_fence_after();
            for (int kb = 0; kb < o.nkb; kb++) {
                bar_wait(smem_u32(&misc.full[s]), ph);
                tc_fence_after();
                const uint32_t a = base + s * stage, b = a + 128 * 128;
                mma_i8_pair_x4(tmem + buf * 256, smem_desc(a, 16, 1024, kLayoutSw128), smem_desc(b, 16, 1024, kLayoutSw128), idesc, kb > 0, smem_u32(&misc.free[s]),
                               kb + 1 == o.nkb ? smem_u32(&misc.d_full[buf]) : 0);
                if (++s == stages) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp >= 4) {
        const int sp = warp & 3, ch = (warp - 4) >> 2, live = o.bsz ? max(0, min(o.T, *o.bsz)) : o.T;
        float* turn = reinterpret_cast<float*>(i8_smem_raw + (base - raw) + kI8Ring + sizeof(Int8GemmMisc)) + (warp - 4) * kI8Turn;
        int it = 0;
        for (int tile = pair; tile < tiles; tile += pairs, it++) {
            int m0, n0;
            place(tile, m0, n0);
            const int buf = it & 1, t = m0 + 32 * sp + lane;
            const uint32_t tcol = tmem + ((uint32_t)(32 * sp) << 16) + buf * 256;
            const float xs = t < o.T ? __ldg(o.xs + t) : 0.f;
            bar_wait(smem_u32(&misc.d_full[buf]), (it >> 1) & 1);
            tc_fence_after();
#pragma unroll 1
            for (int c = 16 * ch; c < bn; c += 64) {
                uint32_t v[16];
                tmem_ld16(tcol + c, v);
                tmem_wait_ld();
                const int n = n0 + c;
                if (n >= o.N) break;
                float f[16];
#pragma unroll
                for (int i = 0; i < 16; i++) f[i] = n + i < o.N ? i8_result((int)v[i], xs, __ldg(o.ws + n + i), o.bias ? __ldg(o.bias + n + i) : 0.f) : 0.f;
                if (TURN) {
                    const int t1 = m0 + 32 * sp + (lane >> 4), col = n + (lane & 15);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 16; i++) turn[33 * i + lane] = f[i];
                    __syncwarp();
#pragma unroll 4
                    for (int k = 0; k < 32; k += 2)
                        if (t1 + k < live && col < o.N) store_hidden(o.y, (long)(t1 + k) * o.y_stride + col, o.type, turn[33 * (lane & 15) + (lane >> 4) + k]);
                } else if (t < live) {
                    const long at = (long)t * o.y_stride + n;
                    if (n + 16 <= o.N) {      // whole sectors of the thread's own row
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; i++) w[i] = __float_as_uint(f[i]);
                        if (o.type != KTB200_TYPE_F32) {
#pragma unroll
                            for (int i = 0; i < 8; i++) w[i] = pack16(f[2 * i], f[2 * i + 1], o.type == KTB200_TYPE_BF16);
                        }
                        uint8_t* y = reinterpret_cast<uint8_t*>(o.y) + at * (o.type == KTB200_TYPE_F32 ? 4 : 2);
                        auto sector = [](uint8_t* to, const uint32_t* u) {
                            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]) : "memory");
                        };
                        sector(y, w);
                        if (o.type == KTB200_TYPE_F32) sector(y + 32, w + 8);
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            if (n + i < o.N) store_hidden(o.y, at + i, o.type, f[i]);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_at(smem_u32(&misc.d_free[buf]), 0)) : "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();      // nobody leaves while the other's copies and products reach for its barriers
    cluster_wait();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// ------------------------------------------------------------------------------------------------ host
static int i8_map(CUtensorMap* map, const void* ptr, int K, long stride, int n, int rows) {      // a box of `rows` x 128 bytes; what lies behind row n or column K comes as zeros
    const EncodeTiledFn enc = encode_tiled();
    if (!enc) { set_error("int8_linear: cuTensorMapEncodeTiled is not available from this driver"); return KTB200_ECUDA; }
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)n}, strides[1] = {(cuuint64_t)stride};
    const cuuint32_t box[2] = {128, (cuuint32_t)rows}, estr[2] = {1, 1};
    const CUresult cr = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS) { set_error("int8_linear: cuTensorMapEncodeTiled failed (%d)", (int)cr); return KTB200_ECUDA; }
    return KTB200_OK;
}
// K splits of int8_rows_kernel: those whose CTAs, two an SM, take least one after the other; kI8Round is what a CTA costs beside its blocks, in blocks
constexpr int kI8Round = 8;
static int i8_splits(long tiles, int nkb, int sms) {
    int best = 1;
    long least = LONG_MAX;
    for (int s = 1; s <= std::min(kI8MaxSplits, nkb); s++) {
        const int per = (nkb + s - 1) / s;
        if ((nkb + per - 1) / per != s) continue;      // (no CTA without a block)
        const long cost = ((tiles * s + 2 * sms - 1) / (2 * sms)) * (per + kI8Round);
        if (cost < least) { least = cost; best = s; }
    }
    return best;
}
template <int NT> static int i8_launch_rows(const void* w, long w_stride, const int8_t* codes, int K, int Kp, const Int8Out& o, int sms, cudaStream_t s) {
    CUtensorMap wmap, xmap;
    int rc = i8_map(&wmap, w, K, w_stride, o.N, 128);
    if (rc == KTB200_OK) rc = i8_map(&xmap, codes, K, Kp, o.T, NT);
    if (rc) return rc;
    const int tiles = (o.N + 127) / 128, tt = (o.T + NT - 1) / NT, splits = i8_splits((long)tiles * tt, o.nkb, sms), per = (o.nkb + splits - 1) / splits;
    KTB_CUDA_CHECK(raise_smem_limit((const void*)int8_rows_kernel<NT>, i8_rows_smem<NT>()));
    cudaLaunchConfig_t lc{};
    lc.gridDim = dim3(tiles, splits, tt);
    lc.blockDim = dim3(kI8RowsThreads);
    lc.dynamicSmemBytes = i8_rows_smem<NT>();
    lc.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1; at[0].val.clusterDim.y = splits; at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = pdl_enabled() ? 2 : 1;
    KTB_CUDA_CHECK(cudaLaunchKernelEx(&lc, int8_rows_kernel<NT>, wmap, xmap, o, per));
    count_launch();
    return KTB200_OK;
}
// Columns of a pair's tile: the multiple of 32 whose rounds take least.  A K block of bn columns takes the larger of its products' time and the shared memory's, in 128 x bn: bn, and about
// 128 + bn / 2; kI8Fixed is what a tile costs beside its blocks, in blocks
constexpr int kI8Fixed = 4;
static int i8_columns(int mt, int N, int nkb, int pairs) {
    int best = 256;
    long least = LONG_MAX;
    for (int bn = 256; bn >= 32; bn -= 32) {
        const long rounds = ((long)mt * ((N + bn - 1) / bn) + pairs - 1) / pairs, cost = rounds * (nkb + kI8Fixed) * std::max(bn, 128 + bn / 2);
        if (cost < least) { least = cost; best = bn; }
    }
    return best;
}
static int i8_launch_gemm(const void* w, long w_stride, const int8_t* codes, int K, int Kp, const Int8Out& o, int sms, cudaStream_t s) {
    const int pairs = sms / 2, mt = (o.T + 255) / 256, bn = i8_columns(mt, o.N, o.nkb, pairs), nt = (o.N + bn - 1) / bn;
    CUtensorMap wmap, xmap;
    int rc = i8_map(&wmap, w, K, w_stride, o.N, bn / 2);
    if (rc == KTB200_OK) rc = i8_map(&xmap, codes, K, Kp, o.T, 128);
    if (rc) return rc;
    const size_t es = type_size(o.type);
    const bool turn = (uintptr_t)o.y % 32 || o.y_stride * es % 32;
    const int smem = turn ? kI8GemmSmemTurn : kI8GemmSmem;
    const auto kernel = turn ? int8_gemm_kernel<true> : int8_gemm_kernel<false>;
    KTB_CUDA_CHECK(raise_smem_limit((const void*)kernel, smem));
    KTB_CUDA_CHECK(launch_pdl(kernel, dim3((unsigned)(2 * std::min<long>((long)mt * nt, pairs))), dim3(kI8GemmThreads), (size_t)smem, s, xmap, wmap, o, bn, mt, nt));
    count_launch();
    return KTB200_OK;
}
template <int TYPE> static cudaError_t i8_launch_quant(const ktb200_int8_linear_params* c, int T, int K, int Kp, int8_t* codes, float* scales, cudaStream_t s) {
    constexpr int E = TYPE == KTB200_TYPE_F32 ? 4 : 8;
    const bool vec = K % E == 0 && ((uintptr_t)c->x & 15) == 0 && c->x_stride % E == 0;
    const int threads = K <= 2048 ? 128 : K <= 8192 ? 256 : 512;
    return launch_pdl(vec ? int8_quant_kernel<TYPE, true> : int8_quant_kernel<TYPE, false>, dim3(T), dim3(threads), (size_t)0, s, c->x, c->x_stride, K, Kp, codes, scales);
}

}  // namespace ktb

using namespace ktb;

extern "C" size_t ktb200_int8_linear_workspace(int n_tokens, int in_features) {
    return n_tokens <= 0 || in_features <= 0 ? 0 : (size_t)n_tokens * (((size_t)in_features + 15) / 16 * 16 + sizeof(float));
}

extern "C" int ktb200_int8_linear(const ktb200_int8_linear_params* c, int n_tokens, void* workspace, size_t workspace_bytes, void* stream) {
    if (!c || c->in_features <= 0 || c->out_features <= 0) { set_error("int8_linear: bad sizes"); return KTB200_EINVAL; }
    if (!is_hidden_type(c->hidden_type)) { set_error("int8_linear: bad hidden_type %d", c->hidden_type); return KTB200_EINVAL; }
    if (c->in_features > INT_MAX / (128 * 128)) { set_error("int8_linear: in_features %d: sums of more than %d products do not fit in 32 bits", c->in_features, INT_MAX / (128 * 128)); return KTB200_EINVAL; }
    if (c->x_stride < c->in_features || c->y_stride < c->out_features || c->weight_stride < c->in_features) { set_error("int8_linear: rows overlap"); return KTB200_EINVAL; }
    if (c->weight_stride % 16 || ((uintptr_t)c->weight & 15)) { set_error("int8_linear: weight rows have to begin at multiples of 16 bytes"); return KTB200_EINVAL; }
    if (n_tokens <= 0) return KTB200_OK;
    if (!c->x || !c->weight || !c->weight_scale || !c->y) { set_error("int8_linear: null pointer"); return KTB200_EINVAL; }
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < ktb200_int8_linear_workspace(n_tokens, c->in_features)) { set_error("int8_linear: workspace missing, too small or not aligned"); return KTB200_EINVAL; }
    const cudaStream_t s = (cudaStream_t)stream;
    int device = 0;
    KTB_CUDA_CHECK(cudaGetDevice(&device));
    const int K = c->in_features, Kp = (K + 15) / 16 * 16, N = c->out_features, T = n_tokens, sms = num_sms(device);
    int8_t* codes = (int8_t*)workspace;
    float* scales = (float*)(codes + (size_t)T * Kp);
    KTB_CUDA_CHECK(c->hidden_type == KTB200_TYPE_F32    ? i8_launch_quant<KTB200_TYPE_F32>(c, T, K, Kp, codes, scales, s)
                   : c->hidden_type == KTB200_TYPE_BF16 ? i8_launch_quant<KTB200_TYPE_BF16>(c, T, K, Kp, codes, scales, s)
                                                        : i8_launch_quant<KTB200_TYPE_F16>(c, T, K, Kp, codes, scales, s));
    count_launch();
    const Int8Out o{scales, c->weight_scale, c->bias, c->y, c->y_stride, c->bsz, c->hidden_type, T, N, (K + 127) / 128};
    auto rows = [&](auto nt) { return i8_launch_rows<decltype(nt)::value>(c->weight, c->weight_stride, codes, K, Kp, o, sms, s); };
    if (T <= 16) return rows(std::integral_constant<int, 16>());
    if (T <= 32) return rows(std::integral_constant<int, 32>());
    if (T <= 64) return rows(std::integral_constant<int, 64>());
    // row tiles whose K is split where the GEMM's narrowest tiles would leave most pairs without one
    if (T <= 128 || (long)((T + 255) / 256) * ((N + 63) / 64) < sms / 2) return rows(std::integral_constant<int, 128>());
    return i8_launch_gemm(c->weight, c->weight_stride, codes, K, Kp, o, sms, s);
}
