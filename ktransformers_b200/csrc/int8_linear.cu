// Linear with 8-bit integers: a scale per token for the activations, a scale per output channel for the weights.
//     s[t] = max_k |x[t][k]| / 127 (fp32),   c[t][k] = rint(x[t][k] / s[t])                     (IEEE quotient; 0 where the row is zero)
//     y[t][n] = cast(float(sum_k c[t][k] w[n][k]) * (s[t] w_scale[n]) + bias[n])                 (the sum in 32-bit integers, exact)
// A row of x with an infinity or NaN has no scale: its results are NaN.
#include <climits>

#include "common.cuh"

namespace ktb {

constexpr int kI8QuantThreads = 256;

// a row per CTA: the largest magnitude, then the codes; codes behind column K (up to Kp) are zeros
__global__ void __launch_bounds__(kI8QuantThreads) int8_quant_kernel(const void* x, int type, long x_stride, int K, int Kp, int8_t* codes, float* scales) {
    __shared__ float red[kI8QuantThreads / 32];
    const long t = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float top = 0.f, odd = 0.f;      // odd: NaN as soon as a value is not finite
    for (int k = threadIdx.x; k < K; k += kI8QuantThreads) {
        const float v = load_hidden(x, t * x_stride + k, type);
        top = fmaxf(top, fabsf(v));
        odd = fmaf(v, 0.f, odd);
    }
    if (odd != odd) top = INFINITY;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) red[warp] = top;
    __syncthreads();
    top = red[0];
#pragma unroll
    for (int w = 1; w < kI8QuantThreads / 32; w++) top = fmaxf(top, red[w]);
    const float s = top == INFINITY ? NAN : __fdiv_rn(top, 127.f);
    for (int k = threadIdx.x; k < Kp; k += kI8QuantThreads) {
        float c = 0.f;
        if (k < K && s > 0.f) c = fminf(fmaxf(rintf(__fdiv_rn(load_hidden(x, t * x_stride + k, type), s)), -127.f), 127.f);
        codes[t * Kp + k] = (int8_t)c;
    }
    if (threadIdx.x == 0) scales[t] = s;
}

// 64 x 64 results of a CTA, 16 bytes of K at a time; a thread has 4 x 4 of them
__global__ void __launch_bounds__(256) int8_tile_kernel(const int8_t* codes, const float* scales, const int8_t* w, const float* w_scale, const float* bias, int T, int K, int Kp, int N, long w_stride,
                                                        void* y, int type, long y_stride, const int* bsz) {
    __shared__ uint32_t xs[64][5], ws[64][5];
    const int live = bsz ? min(T, *bsz) : T, t0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    const int r = threadIdx.x >> 2, c = threadIdx.x & 3;
    for (int k0 = 0; k0 < K; k0 += 16) {
        uint32_t a = 0, b = 0;
        if (t0 + r < T) a = *reinterpret_cast<const uint32_t*>(codes + (long)(t0 + r) * Kp + k0 + 4 * c);
        if (n0 + r < N)
            for (int i = 0; i < 4; i++)
                if (k0 + 4 * c + i < K) b |= (uint32_t)(uint8_t)w[(long)(n0 + r) * w_stride + k0 + 4 * c + i] << (8 * i);
        __syncthreads();
        xs[r][c] = a;
        ws[r][c] = b;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int k = 0; k < 4; k++) acc[i][j] = dp4a_s8s8(xs[ty + 16 * i][k], ws[tx + 16 * j][k], acc[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int t = t0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (t < live && n < N) {
                const float v = (float)acc[i][j] * (scales[t] * w_scale[n]);
                store_hidden(y, (long)t * y_stride + n, type, bias ? v + bias[n] : v);
            }
        }
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
    const int K = c->in_features, Kp = (K + 15) / 16 * 16, N = c->out_features;
    int8_t* codes = (int8_t*)workspace;
    float* scales = (float*)(codes + (size_t)n_tokens * Kp);
    int8_quant_kernel<<<n_tokens, kI8QuantThreads, 0, s>>>(c->x, c->hidden_type, c->x_stride, K, Kp, codes, scales);
    KTB_LAUNCH_CHECK();
    int8_tile_kernel<<<dim3((N + 63) / 64, (n_tokens + 63) / 64), 256, 0, s>>>(codes, scales, (const int8_t*)c->weight, c->weight_scale, c->bias, n_tokens, K, Kp, N, c->weight_stride, c->y,
                                                                              c->hidden_type, c->y_stride, c->bsz);
    KTB_LAUNCH_CHECK();
    return KTB200_OK;
}
