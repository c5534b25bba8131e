// Attention over the paged e4m3 cache on the tensor cores' mma tiles (bf16 queries, head sizes that are multiples of 16 up to 128): decode steps and short portions.
//
// A warp owns 8 or 16 rows = (token, query head) pairs of one portion and one key/value head and takes 16 keys at a time:  S = Q K^T,  t = s log2(e) + log2(value scale),
// p = 2^(t - m),  O += P V,  l += p / (value scale).
// Codes go to m16n8k16 fp16 products as fp16, which holds every e4m3 number exactly (one conversion for two codes), against queries as fp16 too, each row first moved by a power of two so
// that its largest stands below 2^15 (exact for what is within 2^-28 of that), and weights rounded to fp16 (2^-11 of a weight).  (m16n8k32 e4m3 products took more instructions: they
// count as two fp16 ones each, with the conversions of both operands.)
// Key scales multiply scores.  A block's value scale is a power of two in the weight's exponent, so that O needs no scale and the weights of all blocks stand in
// one range: m is 7 below a row's largest t and raised only when a t outgrows it by 15, p <= 2^15.  (With m at that largest the weights beside one key that has most of the weight stood
// among fp16's subnormal numbers: so they are 2^-11 of themselves off down to 2^-21 of the largest, and 2^-32 of that below.)  O / l is the result: 2^m drops out.
//
// The order of a product's sum is free, and taken so that no shuffling is needed: of a key's row, the four threads that share it hold 16 neighbouring bytes each (an S
// step takes 4 of them), and of a value's row each of the eight column groups has its neighbouring bytes, an output tile's columns being dv / 8 apart.
//
// SHARED = false: the CTA's four warps own the same rows and cut the keys among them, tile by tile (decode: a group's heads fill the rows and one pass over the
// keys serves all); each has its own cp.async ring, no barrier in the loop; their sums are joined at the end in shared memory.  TWO: 16 rows, else 8.
// SHARED = true: the warps own 64 rows and share each key tile (16 keys brought by each warp), for portions of many tokens.
#pragma once
#include "mma_tile.cuh"

namespace ktb {

constexpr int kFmThreads = 128, kFmWarps = 4, kFmKeys = 16;
constexpr float kFmTop = 7.f, kFmRaise = 15.f;      // a row's largest weight stands between 2^7 and 2^15 (fp16 holds 2^16 - 2^5)

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two numbers as e4m3 codes (the first in the low byte), and as codes TIMES times what those leave of them
template <int TIMES = 16> __device__ __forceinline__ uint2 split_e4m3(float lo, float hi) {
    const uint32_t first = __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
    const float2 got = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)first, __NV_E4M3)));
    return make_uint2(first, __nv_cvt_float2_to_fp8x2(make_float2((lo - got.x) * TIMES, (hi - got.y) * TIMES), __NV_SATFINITE, __NV_E4M3));
}
// two e4m3 codes (the low half of a word) as two fp16 numbers
__device__ __forceinline__ uint32_t f16_of_codes(uint32_t two) {
    uint32_t r;
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %1;\ncvt.rn.f16x2.e4m3x2 %0, l;\n}" : "=r"(r) : "r"(two));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void cp_async_bytes16(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_bytes8(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(ok ? 8 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}

// heads of a group that one warp's rows take: the largest divisor of the group up to 16
__host__ __device__ inline int fm_heads(int R) {
    for (int h = R < 16 ? R : 16; h > 1; h--)
        if (R % h == 0) return h;
    return 1;
}
// shared memory of a 16-key tile: keys, values, (key scale, value scale) per key
template <int DP, int DVP> constexpr int fm_tile_bytes() { return kFmKeys * (DP + DVP) + kFmKeys * 8; }
template <bool SHARED> constexpr int fm_stages() { return SHARED ? 3 : 4; }
template <int DP, int DVP, bool SHARED> constexpr int fm_smem() {
    const int ring = kFmWarps * fm_stages<SHARED>() * fm_tile_bytes<DP, DVP>(), join = kFmWarps * 16 * (DVP + 4) * 4;
    return ring > join || SHARED ? ring : join;
}

template <int DP, int DVP, bool SHARED, bool TWO> __global__ void __launch_bounds__(kFmThreads, 3) fp8_attn_mma_kernel(const Fp8Attn a, int RH) {
    constexpr int KC = DP / 64, VB = DVP / 8, TILE = fm_tile_bytes<DP, DVP>(), STAGES = fm_stages<SHARED>(), NT = DVP / 8, ROWS = TWO ? 2 : 1;
    extern __shared__ __align__(16) unsigned char fm_smem_raw[];
    __shared__ int info[6];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gq = lane >> 2, tq = lane & 3;
    const int d = a.d, dv = a.dv, ps = a.pages.page_size, TOKS = 8 * ROWS / RH, CTOKS = a.ctoks, R = a.H / a.G, hblocks = R / RH;
    const uint32_t smem = (uint32_t)__cvta_generic_to_shared(fm_smem_raw);
    griddep_launch_dependents();
    griddep_wait();
    if (warp == 0) fp8_find_tokens(a, blockIdx.x, CTOKS, info);
    // columns behind a head's last are zeros throughout
    if (d < DP || dv < DVP)
        for (int i = tid; i < kFmWarps * STAGES * TILE / 16; i += kFmThreads) reinterpret_cast<uint4*>(fm_smem_raw)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const int tok0 = info[0], ntok = info[1], pos0 = info[2], slot = info[3];
    if (ntok <= 0) return;
    const int g = blockIdx.y / hblocks, h0 = g * R + (blockIdx.y % hblocks) * RH, max_pos = pos0 + ntok - 1;
    // the key range of the CTA's tokens, in parts that begin at multiples of 16
    const int lo = fp8_first_visible(pos0, a.window, a.chunk), lo16 = lo & ~(kFmKeys - 1);
    constexpr int STEP = kFmWarps * kFmKeys;
    const bool cut = a.part > 0 && max_pos + 1 - lo16 > a.part;
    const int k_lo = lo16 + blockIdx.z * a.part, k_hi = cut ? min(max_pos + 1, k_lo + a.part) : max_pos + 1;
    if (k_lo >= k_hi) return;
    // this thread's rows
    const int wtok = SHARED ? warp * TOKS : 0, rows = TOKS * RH;
    const int tokA = wtok + gq / RH, tokB = wtok + (gq + 8) / RH, hA = h0 + gq % RH, hB = h0 + (gq + 8) % RH;
    const bool vA = gq < rows && tokA < ntok, vB = TWO && gq + 8 < rows && tokB < ntok;
    const int pA = pos0 + tokA, pB = pos0 + tokB, fA = fp8_first_visible(pA, a.window, a.chunk), fB = fp8_first_visible(pB, a.window, a.chunk);
    float O[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++) O[n][e] = 0.f;
    float mA = -INFINITY, mB = -INFINITY, lA = 0.f, lB = 0.f;
    {
        // ---------------------------------------------------------------- the ring: a tile is 16 keys from a multiple of 16 on
        const bool slot_ok = (unsigned)slot < (unsigned)a.pages.slots, whole = ps % kFmKeys == 0;
        const int* pt = a.pages.table + (slot_ok ? (long)slot * a.pages.max_pages : 0);
        const uint32_t ring = smem + warp * STAGES * TILE;
        const int piece = lane & 7, r4 = lane >> 3;      // eight neighbouring lanes bring a row's 128 bytes
        // the page of the tile (or of the lane's row in it) that is brought next, looked up a tile ahead, and the row in that page
        int page = -1, off = 0, logical = 0, col = 0;
        auto look = [&](int k0) {
            const int kp = whole ? k0 : k0 + (lane & 15);
            page = -1;
            if (kp >= k_hi || !slot_ok) return;
            if (!whole) { logical = kp / ps; off = kp - logical * ps; col = logical % a.pages.max_pages; }
            page = pt[col];
            if ((unsigned)page >= (unsigned)a.pages.n_pages) page = -1;
        };
        auto load_tile = [&](int stage, int k0) {      // this warp's 16 keys from k0 on
            if (k0 < k_hi) {
                const uint32_t kd = ring + stage * TILE, vd = kd + kFmKeys * DP, sd = vd + kFmKeys * DVP;
                const long block = (long)page * a.G + g, row0 = block * ps + off;
                // (keys that no row sees may be anything, NaN too: they come as zeros, and so do those of pages that are not there)
                const bool full = whole && k0 >= lo && k0 + kFmKeys <= k_hi && page >= 0;
                const int r16 = lane & 15;
                const bool ok16 = page >= 0 && k0 + r16 < k_hi && k0 + r16 >= lo;
                if (lane < 16) cp_async_bytes8(sd + 8 * r16, ok16 ? a.scales + 2 * block : a.scales, ok16);
                // a key row's chunks change halves in odd rows, a value row's by its number: no two of the lanes that read together meet in a bank
                const uint32_t kx = 16 * (DP == 128 ? piece ^ ((r4 & 1) << 2) : piece);
                if (full) {
                    const uint8_t *k = a.k_codes + (row0 + r4) * d + 16 * piece, *v = a.v_codes + (row0 + r4) * dv + 16 * piece;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int r = 4 * i + r4;
                        if (16 * piece < d) cp_async_bytes16(kd + r * DP + kx, k + 4 * i * d, true);
                        if (16 * piece < dv) cp_async_bytes16(vd + r * DVP + 16 * (DVP == 128 ? piece ^ (r & 7) : piece ^ ((r >> 1) & 3)), v + 4 * i * dv, true);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int r = 4 * i + r4;
                        const long row = whole ? row0 + r : __shfl_sync(0xffffffffu, row0, r);
                        const bool ok = (whole ? page : __shfl_sync(0xffffffffu, page, r)) >= 0 && k0 + r < k_hi && k0 + r >= lo;
                        if (16 * piece < d) cp_async_bytes16(kd + r * DP + kx, ok ? a.k_codes + row * d + 16 * piece : a.k_codes, ok);
                        if (16 * piece < dv) cp_async_bytes16(vd + r * DVP + 16 * (DVP == 128 ? piece ^ (r & 7) : piece ^ ((r >> 1) & 3)), ok ? a.v_codes + row * dv + 16 * piece : a.v_codes, ok);
                    }
                }
                if (whole) {
                    off += STEP;
                    while (off >= ps) {
                        off -= ps;
                        if (++col == a.pages.max_pages) col = 0;
                    }
                }
                look(k0 + STEP);
            }
            cp_async_commit();
        };
        if (whole) {
            const int k0 = k_lo + warp * kFmKeys;
            logical = k0 / ps; off = k0 - logical * ps; col = logical % a.pages.max_pages;
        }
        look(k_lo + warp * kFmKeys);
#pragma unroll
        for (int i = 0; i < STAGES - 1; i++) load_tile(i, k_lo + warp * kFmKeys + i * STEP);
        // ---------------------------------------------------------------- queries: the thread's 16 columns of every 64
        uint32_t Q[ROWS][8 * KC];
        float fac[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; r++) {
            const bool v = r ? vB : vA;
            const __nv_bfloat16* row = (const __nv_bfloat16*)a.q + ((long)(tok0 + (r ? tokB : tokA)) * a.H + (r ? hB : hA)) * d;
            uint32_t(&w)[8 * KC] = Q[r];
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int at = 64 * c + 16 * tq + 8 * i;
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (v && at < d) x = *reinterpret_cast<const uint4*>(row + at);
                    w[8 * c + 4 * i] = x.x; w[8 * c + 4 * i + 1] = x.y; w[8 * c + 4 * i + 2] = x.z; w[8 * c + 4 * i + 3] = x.w;
                }
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 8 * KC; i++) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^(14 - e) of a largest 1.f 2^e, within what fp32 holds with its inverse (an infinity stays one)
            const int up = min(126, max(-112, 14 - ((int)(__float_as_uint(top) >> 23) - 127)));
            const float by = __uint_as_float((uint32_t)(up + 127) << 23);
            fac[r] = v ? (a.head_scale ? a.scale * a.head_scale[r ? hB : hA] : a.scale) / by * (a.softcap > 0.f ? 1.f : kLog2e) : 0.f;
#pragma unroll
            for (int i = 0; i < 8 * KC; i++) w[i] = pack_f16(__uint_as_float(w[i] << 16) * by, __uint_as_float(w[i] & 0xffff0000u) * by);
        }
        const float two_over_cap = a.softcap > 0.f ? 2.0f / a.softcap : 0.f;
        const int w_min_pos = pos0 + wtok, w_max_pos = pos0 + min(ntok - 1, wtok + TOKS - 1);
        const int w_first = fp8_first_visible(w_min_pos, a.window, a.chunk), w_last_first = fp8_first_visible(w_max_pos, a.window, a.chunk);
        // ---------------------------------------------------------------- one tile of 16 keys
        auto take = [&](uint32_t kd, int k0) {
            const uint32_t vd = kd + kFmKeys * DP, sd = vd + kFmKeys * DVP;
            float S[2][4];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int r = 8 * n + gq;
#pragma unroll
                for (int e = 0; e < 4; e++) S[n][e] = 0.f;
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    const uint4 k = lds16(kd + r * DP + 16 * (DP == 128 ? (4 * c + tq) ^ ((r & 1) << 2) : tq));
                    const uint32_t kw[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
                    for (int s = 0; s < 4; s++) {      // columns 4 s .. 4 s + 3 of the thread's 16
                        const int at = 8 * c + 2 * s;
                        const uint32_t q[4] = {Q[0][at], TWO ? Q[ROWS - 1][at] : 0u, Q[0][at + 1], TWO ? Q[ROWS - 1][at + 1] : 0u};
                        mma_f16_16816(S[n], q, f16_of_codes(kw[s]), f16_of_codes(kw[s] >> 16));
                    }
                }
            }
            // the thread's keys: k0 + 8 n + 2 tq + {0, 1}
            float inv[4];
            const bool plain = k0 + kFmKeys - 1 <= w_min_pos && k0 >= w_last_first && k0 + kFmKeys <= k_hi;
            float top[ROWS];
#pragma unroll
            for (int h = 0; h < ROWS; h++) top[h] = -INFINITY;
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const uint4 sc = lds16(sd + 8 * (8 * n + 2 * tq));
                const float ks[2] = {__uint_as_float(sc.x), __uint_as_float(sc.z)};
                const uint32_t vs[2] = {sc.y, sc.w};
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int key = k0 + 8 * n + 2 * tq + i;
                    const float ve = (float)((int)(vs[i] >> 23) - 127);
                    inv[2 * n + i] = vs[i] ? __uint_as_float((254u << 23) - vs[i]) : 0.f;      // 1 / value scale (a page that is not there: scales of zero)
#pragma unroll
                    for (int h = 0; h < ROWS; h++) {
                        float x = S[n][2 * h + i] * (fac[h] * ks[i]);
                        if (a.softcap > 0.f) x = a.softcap * kLog2e * (1.0f - __fdividef(2.0f, __expf(x * two_over_cap) + 1.0f));      // c tanh(s / c): a few 1e-7 of the cap off
                        x += ve;
                        if (!plain && !((h ? vB : vA) && key <= (h ? pB : pA) && key >= (h ? fB : fA) && key < k_hi)) x = -INFINITY;
                        if (vs[i] == 0) x = -INFINITY;
                        S[n][2 * h + i] = x;
                        top[h] = fmaxf(top[h], x);
                    }
                }
            }
            bool raise[ROWS], any = false;
#pragma unroll
            for (int h = 0; h < ROWS; h++) {
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                const float m = h ? mB : mA;
                raise[h] = top[h] > m + kFmRaise || (m == -INFINITY && top[h] > -INFINITY);
                any |= raise[h];
            }
            if (__any_sync(0xffffffffu, any)) {
#pragma unroll
                for (int h = 0; h < ROWS; h++) {
                    float &m = h ? mB : mA, &l = h ? lB : lA;
                    const float k = raise[h] ? exp2_approx(m - (top[h] - kFmTop)) : 1.f;      // (2^-inf = 0: nothing was summed yet)
                    if (raise[h]) m = top[h] - kFmTop;
                    l *= k;
#pragma unroll
                    for (int n = 0; n < NT; n++) { O[n][2 * h] *= k; O[n][2 * h + 1] *= k; }
                }
            }
#pragma unroll
            for (int h = 0; h < ROWS; h++) {
                const float m = h ? mB : mA, u = m == -INFINITY ? 0.f : m;
                float &l = h ? lB : lA;
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        S[n][2 * h + i] = exp2_approx(S[n][2 * h + i] - u);
                        l = fmaf(S[n][2 * h + i], inv[2 * n + i], l);
                    }
            }
            const uint32_t P[4] = {pack_f16(S[0][0], S[0][1]), TWO ? pack_f16(S[0][2], S[0][3]) : 0u, pack_f16(S[1][0], S[1][1]), TWO ? pack_f16(S[1][2], S[1][3]) : 0u};
            // values: rows 2 tq, 2 tq + 1 and 8 more, the VB bytes of column group gq
            uint32_t v[4][VB / 4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = 2 * tq + (i & 1) + 8 * (i >> 1);
                if constexpr (VB == 16) {
                    const uint4 x = lds16(vd + r * DVP + 16 * (gq ^ (r & 7)));
                    v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
                } else {
                    const uint2 x = lds8(vd + r * DVP + 16 * ((gq >> 1) ^ ((r >> 1) & 3)) + 8 * (gq & 1));
                    v[i][0] = x.x; v[i][1] = x.y;
                }
            }
            if (!plain) {      // a value that is NaN belongs to the rows that see it: 0 x NaN would give it to the others
                uint32_t odd = 0;
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int w = 0; w < VB / 4; w++) odd |= (v[i][w] & 0x7f7f7f7fu) + 0x01010101u;
                if (__any_sync(0xffffffffu, odd & 0x80808080u)) {
#pragma unroll 1
                    for (int r = 0; r < kFmKeys; r++) {
                        const int key = k0 + r;
                        const bool seeA = vA && key <= pA && key >= fA, seeB = vB && key <= pB && key >= fB;
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const int grp = 2 * tq + c;
#pragma unroll
                            for (int n = 0; n < NT; n++) {
                                const uint32_t at = vd - smem + r * DVP + (VB == 16 ? 16 * (grp ^ (r & 7)) : 16 * ((grp >> 1) ^ ((r >> 1) & 3)) + 8 * (grp & 1)) + n;
                                const bool bad = (fm_smem_raw[at] & 0x7f) == 0x7f;
                                if (bad && seeA) O[n][c] = NAN;
                                if (TWO && bad && seeB) O[n][2 + c] = NAN;
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int w = 0; w < VB / 4; w++) v[i][w] &= ~(((((v[i][w] & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u) * 0xffu);
                }
            }
#pragma unroll
            for (int w = 0; w < VB / 4; w++) {
#pragma unroll
                for (int h = 0; h < 2; h++) {      // columns 4 w + 2 h, 4 w + 2 h + 1
                    const uint32_t x = __byte_perm(v[0][w], v[1][w], h ? 0x7362 : 0x5140), y = __byte_perm(v[2][w], v[3][w], h ? 0x7362 : 0x5140);
                    mma_f16_16816(O[4 * w + 2 * h], P, f16_of_codes(x), f16_of_codes(y));
                    mma_f16_16816(O[4 * w + 2 * h + 1], P, f16_of_codes(x >> 16), f16_of_codes(y >> 16));
                }
            }
        };
        // ---------------------------------------------------------------- the loop
        int stage = 0;
        for (int j0 = k_lo; j0 < k_hi; j0 += STEP) {
            cp_async_wait<STAGES - 2>();
            if (SHARED) __syncthreads(); else __syncwarp();      // the tile is here for all who read it, and nobody reads the stage that is filled next
            load_tile((stage + STAGES - 1) % STAGES, j0 + warp * kFmKeys + (STAGES - 1) * STEP);
            if (SHARED) {
                for (int w = 0; w < kFmWarps; w++) {
                    const int k0 = j0 + w * kFmKeys;
                    if (k0 >= k_hi || wtok >= ntok || k0 > w_max_pos || k0 + kFmKeys <= w_first) continue;
                    take(smem + (w * STAGES + stage) * TILE, k0);
                }
            } else {
                const int k0 = j0 + warp * kFmKeys;
                if (k0 < k_hi) take(ring + stage * TILE, k0);
            }
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        cp_async_wait<0>();
    }
    lA += __shfl_xor_sync(0xffffffffu, lA, 1);
    lA += __shfl_xor_sync(0xffffffffu, lA, 2);
    lB += __shfl_xor_sync(0xffffffffu, lB, 1);
    lB += __shfl_xor_sync(0xffffffffu, lB, 2);
    // thread (gq, tq) has of row gq (and gq + 8) the columns 2 tq VB + n (O[n][0]) and (2 tq + 1) VB + n (O[n][1])
    if (!SHARED) {      // the warps' sums: each row's largest reference, then every thread some of the columns
        float* join = reinterpret_cast<float*>(fm_smem_raw);      // [warp][16][DVP + 4]: maximum, sum, columns
        __syncthreads();
        constexpr int LD = DVP + 4;
#pragma unroll
        for (int r = 0; r < 2; r++) {
            if (r && !TWO) break;
            float* o = join + ((long)warp * 16 + gq + 8 * r) * LD;
            if (tq == 0) { o[0] = r ? mB : mA; o[1] = r ? lB : lA; }
#pragma unroll
            for (int n = 0; n < NT; n += 4)
#pragma unroll
                for (int c = 0; c < 2; c++)
                    *reinterpret_cast<float4*>(o + 4 + (2 * tq + c) * VB + n) = make_float4(O[n][2 * r + c], O[n + 1][2 * r + c], O[n + 2][2 * r + c], O[n + 3][2 * r + c]);
        }
        __syncthreads();
        // a row per group of eight threads
        for (int r = tid >> 3; r < rows; r += kFmThreads / 8) {
            const int tok = r / RH, h = h0 + r % RH;
            if (tok >= ntok) continue;
            float m = -INFINITY, l = 0.f, wgt[kFmWarps];
#pragma unroll
            for (int w = 0; w < kFmWarps; w++) m = fmaxf(m, join[(w * 16 + r) * LD]);
#pragma unroll
            for (int w = 0; w < kFmWarps; w++) {
                const float mw = join[(w * 16 + r) * LD];
                wgt[w] = mw == -INFINITY ? 0.f : exp2_approx(mw - m);
                l = fmaf(wgt[w], join[(w * 16 + r) * LD + 1], l);
            }
            const long row = (long)(tok0 + tok) * a.H + h;
            float* part = cut ? a.partial + (row * a.parts + blockIdx.z) * (dv + 2) : nullptr;
            float inv = 1.f;
            if (part) {
                if ((tid & 7) == 0) { part[0] = m; part[1] = l; }
            } else {
                if (a.sink) {
                    const float k = fp8_sink(a.sink[h], m, l);
#pragma unroll
                    for (int w = 0; w < kFmWarps; w++) wgt[w] *= k;
                }
                inv = l > 0.f || l != l ? a.out_scale / l : 0.f;
            }
            __nv_bfloat16* out = (__nv_bfloat16*)a.out + (long)(tok0 + tok) * a.out_stride + (long)h * dv;
            for (int c = (tid & 7) * 4; c < dv; c += 32) {
                float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kFmWarps; w++) {
                    const float4 x = *reinterpret_cast<const float4*>(join + (w * 16 + r) * LD + 4 + c);
                    s.x = fmaf(wgt[w], x.x, s.x); s.y = fmaf(wgt[w], x.y, s.y); s.z = fmaf(wgt[w], x.z, s.z); s.w = fmaf(wgt[w], x.w, s.w);
                }
                if (part) {
                    *reinterpret_cast<float2*>(part + 2 + c) = make_float2(s.x, s.y);
                    *reinterpret_cast<float2*>(part + 4 + c) = make_float2(s.z, s.w);
                } else {
                    const uint32_t u = pack_bf16(s.x * inv, s.y * inv), v = pack_bf16(s.z * inv, s.w * inv);
                    if (((reinterpret_cast<uintptr_t>(out) & 7) == 0)) {
                        *reinterpret_cast<uint2*>(out + c) = make_uint2(u, v);
                    } else {
                        const uint16_t b[4] = {(uint16_t)u, (uint16_t)(u >> 16), (uint16_t)v, (uint16_t)(v >> 16)};
#pragma unroll
                        for (int i = 0; i < 4; i++) reinterpret_cast<uint16_t*>(out)[c + i] = b[i];
                    }
                }
            }
        }
        return;
    }
#pragma unroll
    for (int r = 0; r < 2; r++) {
        if (!(r ? vB : vA)) continue;
        const int tok = r ? tokB : tokA, h = r ? hB : hA;
        float m = r ? mB : mA, l = r ? lB : lA, k = 1.f;
        const long row = (long)(tok0 + tok) * a.H + h;
        float* part = cut ? a.partial + (row * a.parts + blockIdx.z) * (dv + 2) : nullptr;
        if (part) {
            if (tq == 0) { part[0] = m; part[1] = l; }
        } else {
            if (a.sink) k = fp8_sink(a.sink[h], m, l);
            k = l > 0.f || l != l ? k * a.out_scale / l : 0.f;
        }
        __nv_bfloat16* out = (__nv_bfloat16*)a.out + (long)(tok0 + tok) * a.out_stride + (long)h * dv;
        const bool vec = (reinterpret_cast<uintptr_t>(out) & 7) == 0;
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int n = 0; n < NT; n += 4) {
                const int col = (2 * tq + c) * VB + n;
                if (col >= dv) continue;
                const float s0 = O[n][2 * r + c] * k, s1 = O[n + 1][2 * r + c] * k, s2 = O[n + 2][2 * r + c] * k, s3 = O[n + 3][2 * r + c] * k;
                if (part) {
                    *reinterpret_cast<float2*>(part + 2 + col) = make_float2(s0, s1);
                    *reinterpret_cast<float2*>(part + 4 + col) = make_float2(s2, s3);
                } else if (vec) {
                    *reinterpret_cast<uint2*>(out + col) = make_uint2(pack_bf16(s0, s1), pack_bf16(s2, s3));
                } else {
                    const uint32_t u = pack_bf16(s0, s1), v = pack_bf16(s2, s3);
                    const uint16_t b[4] = {(uint16_t)u, (uint16_t)(u >> 16), (uint16_t)v, (uint16_t)(v >> 16)};
#pragma unroll
                    for (int i = 0; i < 4; i++) reinterpret_cast<uint16_t*>(out)[col + i] = b[i];
                }
            }
    }
}

// whether these tiles take the call
static bool fm_takes(const ktb200_fp8_attn_params* c, int dtype) {
    return dtype == KTB200_TYPE_BF16 && c->dim % 16 == 0 && c->vdim % 16 == 0 && c->dim <= 128 && c->vdim <= 128 &&
           ((reinterpret_cast<uintptr_t>(c->q) | reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->v_codes)) & 15) == 0 && (reinterpret_cast<uintptr_t>(c->scales) & 7) == 0;
}
// Which form: 64 rows that share key tiles where portions have more tokens than two 16-row tiles take; else 8 rows a tile where those hold a portion's tokens, 16 where not
struct FmForm { int RH, toks; bool shared, two; };
static FmForm fm_form(const ktb200_fp8_attn_params* c, int n_tokens) {
    FmForm f;
    f.RH = fm_heads(c->heads / c->kv_heads);
    f.shared = (long)n_tokens > 2L * c->n_seqs * (16 / f.RH);
    f.two = f.shared || f.RH > 8 || (long)n_tokens > (long)c->n_seqs * (8 / f.RH);
    f.toks = (f.shared ? kFmWarps : 1) * ((f.two ? 16 : 8) / f.RH);
    return f;
}
template <int DP, int DVP, bool SHARED, bool TWO> static cudaError_t fm_launch_as(const Fp8Attn& a, int RH, dim3 grid, cudaStream_t s) {
    constexpr int smem = fm_smem<DP, DVP, SHARED>();
    const cudaError_t e = raise_smem_limit((const void*)fp8_attn_mma_kernel<DP, DVP, SHARED, TWO>, smem);
    return e != cudaSuccess ? e : launch_pdl(fp8_attn_mma_kernel<DP, DVP, SHARED, TWO>, grid, dim3(kFmThreads), (size_t)smem, s, a, RH);
}
template <bool SHARED, bool TWO> static cudaError_t fm_launch_of(const Fp8Attn& a, int RH, dim3 grid, cudaStream_t s) {
    if (a.d <= 64) return a.dv <= 64 ? fm_launch_as<64, 64, SHARED, TWO>(a, RH, grid, s) : fm_launch_as<64, 128, SHARED, TWO>(a, RH, grid, s);
    return a.dv <= 64 ? fm_launch_as<128, 64, SHARED, TWO>(a, RH, grid, s) : fm_launch_as<128, 128, SHARED, TWO>(a, RH, grid, s);
}
static cudaError_t fm_launch(const Fp8Attn& a, const FmForm& f, dim3 grid, cudaStream_t s) {
    return f.shared ? fm_launch_of<true, true>(a, f.RH, grid, s) : f.two ? fm_launch_of<false, true>(a, f.RH, grid, s) : fm_launch_of<false, false>(a, f.RH, grid, s);
}

}  // namespace ktb
