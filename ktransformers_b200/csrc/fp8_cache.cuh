// The paged e4m3 cache: what its append (fp8_cache.cu) and its attention (fp8_attn.cu) share.
//
// A page holds page_size tokens of every key/value head, head by head: keys [pages][G][page_size][d], values [pages][G][page_size][dv], one byte each, and
// scales [pages][G][2] (fp32: keys, values).  A block is one head of one page; what it holds stands for code * scale.  Scales are powers of two, 2^e with the smallest
// e in [-64, 64] for which 448 2^e reaches every value of the block (448: e4m3's largest), so that
//   - a block whose later tokens are larger is re-scaled by moving its codes' exponents, exactly but for what becomes subnormal;
//   - code * scale is exact in bf16 and fp32, codes alone are exact in fp16;
//   - the attention takes a block's value scale into the exponent of its weights.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"
#include "seq_common.cuh"

namespace ktb {

constexpr int kFp8EMin = -64, kFp8EMax = 64;

// the page of position p of the sequence in table row `slot` (the row is a ring), or -1 where there is none
struct Fp8Pages {
    const int* table;
    int slots, max_pages, page_size, n_pages;
    __device__ __forceinline__ int page(int slot, int logical) const {
        if ((unsigned)slot >= (unsigned)slots) return -1;
        const int p = table[(long)slot * max_pages + logical % max_pages];
        return (unsigned)p < (unsigned)n_pages ? p : -1;
    }
};

// Which of the step's portions item b belongs to, and which of the portion's items it is, where portion s has count(s) of them (called by a whole warp): false where
// there is no such item.  The counts of 32 portions are made side by side, so that a step of hundreds of them costs a few loads one after the other and not hundreds.
template <typename Count> __device__ __forceinline__ bool fp8_find(int b, int n_seqs, Count count, int& seq, int& item) {
    const int lane = threadIdx.x & 31;
    for (int s0 = 0; s0 < n_seqs; s0 += 32) {
        const int n = s0 + lane < n_seqs ? count(s0 + lane) : 0;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned has = __ballot_sync(0xffffffffu, b < sum);
        if (has) {
            const int at = __ffs(has) - 1;
            seq = s0 + at;
            item = b - __shfl_sync(0xffffffffu, sum - n, at);
            return true;
        }
        b -= __shfl_sync(0xffffffffu, sum, 31);
    }
    return false;
}

}  // namespace ktb
