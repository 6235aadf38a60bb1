// Products in 8-bit integers: y[m][n] = sx[m] sw[n] sum_k qx[m][k] qw[n][k] (+ bias[n]) (GELU), qx / qw symmetric 8-bit values with one
// scale per row (token, output channel): q = 127 x / max |x| rounded to the nearest (ties to even), scale = max |x| / 127.
//
// The sum is an integer and exact (127^2 K < 2^31 bounds K at 131,072); it becomes f32 (2^-24) before the two scales.  A row whose values
// are not all finite has a scale that is not finite and gives NaN; a row of zeros gives the bias.
// Bound: the integer matrix cores (twice the bf16 rate) for many rows, HBM (the weights once, half the bf16 bytes) for few.
#include "gemm_common.h"

namespace {

inline int ok() { return hipGetLastError() == hipSuccess ? MMSUM_OK : MMSUM_ERR_HIP; }
typedef int i32x4_t __attribute__((ext_vector_type(4)));

// ---- quantisation: one workgroup a row ---------------------------------------------------------------------------------------------
// 127 x first, so that x = max / 2 lands on the tie it is; rows near the end of the f32 range are taken down by 2^8 before that
__device__ __forceinline__ float row_pre(float top) { return top > 0x1p119f ? 0x1p-8f : 1.f; }
__device__ __forceinline__ int quantize(float x, float pre, float top_pre) {
    const float q = rintf((x * pre) * 127.f / top_pre);
    return q == q ? (int)fminf(fmaxf(q, -127.f), 127.f) : 0;
}

template <typename T>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ x, long ldx, int K, int8_t* __restrict__ q, long ldq, float* __restrict__ scale) {
    __shared__ float sh[4];
    __shared__ int bad[4];
    const long row = blockIdx.x;
    const int tid = threadIdx.x;
    float top = 0.f;
    int nan = 0;
    for (int k = tid; k < K; k += 256) {
        const float v = to_f32(x[row * ldx + k]);
        top = fmaxf(top, fabsf(v));
        nan |= v != v;
    }
    top = warp_max(top);
    const bool wave_nan = __any(nan);
    if ((tid & 63) == 0) { sh[tid >> 6] = top; bad[tid >> 6] = wave_nan; }
    __syncthreads();
    top = fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
    if (bad[0] | bad[1] | bad[2] | bad[3]) top = NAN;
    const float pre = row_pre(top), tp = top * pre;
    for (int k = tid; k < (int)ldq; k += 256) q[row * ldq + k] = k < K ? (int8_t)quantize(to_f32(x[row * ldx + k]), pre, tp) : (int8_t)0;
    if (tid == 0) scale[row] = top / 127.f;
}

// ---- product -----------------------------------------------------------------------------------------------------------------------
struct I8Args {
    const int8_t* A; long lda; const float* sa; const int8_t* B; long ldb; const float* sb; const float* bias;
    void* C; long ldc; int M, N, K, gelu;
};

// v_mfma_i32_16x16x64_i8: lane l holds 16 consecutive k of row l & 15, k group l >> 4; result column l & 15, rows 4 (l >> 4) + e
template <typename T>
__global__ __launch_bounds__(256) void gemm_i8_kernel(I8Args p) {
    __shared__ __attribute__((aligned(16))) int8_t sA[64 * 64], sB[64 * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long m0 = (long)blockIdx.y * 64, n0 = (long)blockIdx.x * 64;
    i32x4_t acc[4] = {};
    for (int k0 = 0; k0 < p.K; k0 += 64) {
        const int r = tid >> 2, ch = tid & 3;
        const long am = m0 + r < p.M ? m0 + r : p.M - 1, bn = n0 + r < p.N ? n0 + r : p.N - 1;
        const u32x4_t va = *reinterpret_cast<const u32x4_t*>(p.A + am * p.lda + k0 + ch * 16), vb = *reinterpret_cast<const u32x4_t*>(p.B + bn * p.ldb + k0 + ch * 16);
        __syncthreads();
        *reinterpret_cast<u32x4_t*>(sA + r * 64 + ch * 16) = va;
        *reinterpret_cast<u32x4_t*>(sB + r * 64 + ch * 16) = vb;
        __syncthreads();
        const i32x4_t a = *reinterpret_cast<const i32x4_t*>(sA + (wave * 16 + (lane & 15)) * 64 + (lane >> 4) * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const i32x4_t b = *reinterpret_cast<const i32x4_t*>(sB + (j * 16 + (lane & 15)) * 64 + (lane >> 4) * 16);
            acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc[j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const long m = m0 + wave * 16 + 4 * (lane >> 4) + e, n = n0 + j * 16 + (lane & 15);
            if (m < p.M && n < p.N) {
                float v = (float)acc[j][e] * p.sa[m] * p.sb[n];
                if (p.bias) v += p.bias[n];
                if (p.gelu) v = gelu_f(v);
                static_cast<T*>(p.C)[m * p.ldc + n] = from_f32<T>(v);
            }
        }
}

}  // namespace

extern "C" int mmsum_quantize_i8(int dtype, const void* x, long ldx, int M, int K, void* q, long ldq, float* scale, void* stream) {
    if (M <= 0 || K <= 0 || ldx < K || ldq < K || ldq % 64 || ldq > 0x7fffffc0L) return MMSUM_ERR_BAD_SHAPE;
    if (dtype != MMSUM_BF16 && dtype != MMSUM_F32) return MMSUM_ERR_BAD_DTYPE;
    if (((uintptr_t)q & 15) || ((uintptr_t)x & (dtype == MMSUM_BF16 ? 1 : 3))) return MMSUM_ERR_BAD_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MMSUM_BF16) hipLaunchKernelGGL((quantize_kernel<bf16_t>), dim3(M), dim3(256), 0, s, (const bf16_t*)x, ldx, K, (int8_t*)q, ldq, scale);
    else hipLaunchKernelGGL((quantize_kernel<float>), dim3(M), dim3(256), 0, s, (const float*)x, ldx, K, (int8_t*)q, ldq, scale);
    return ok();
}

extern "C" int mmsum_gemm_i8(const void* qx, long ldx, const float* sx, const void* qw, long ldw, const float* sw, const float* bias, int dtype_out, void* y, long ldy,
                             int M, int N, int K, int gelu, void* stream) {
    if (M <= 0 || N <= 0 || K <= 0 || K % 64 || K > 131072 || ldx < K || ldw < K || ldx % 16 || ldw % 16 || ldy < N) return MMSUM_ERR_BAD_SHAPE;
    if (dtype_out != MMSUM_BF16 && dtype_out != MMSUM_F32) return MMSUM_ERR_BAD_DTYPE;
    if ((((uintptr_t)qx | (uintptr_t)qw) & 15) || ((uintptr_t)y & (dtype_out == MMSUM_BF16 ? 1 : 3))) return MMSUM_ERR_BAD_ALIGN;
    I8Args p = {static_cast<const int8_t*>(qx), ldx, sx, static_cast<const int8_t*>(qw), ldw, sw, bias, y, ldy, M, N, K, gelu};
    const dim3 grid((unsigned)((N + 63) / 64), (unsigned)((M + 63) / 64));
    if (grid.y > 65535) return MMSUM_ERR_BAD_SHAPE;
    if (dtype_out == MMSUM_BF16) hipLaunchKernelGGL((gemm_i8_kernel<bf16_t>), grid, dim3(256), 0, (hipStream_t)stream, p);
    else hipLaunchKernelGGL((gemm_i8_kernel<float>), grid, dim3(256), 0, (hipStream_t)stream, p);
    return ok();
}
