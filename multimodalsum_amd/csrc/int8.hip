// Products in 8-bit integers: y[m][n] = sx[m] sw[n] sum_k qx[m][k] qw[n][k] (+ bias[n]) (GELU), qx / qw symmetric 8-bit values with one
// scale per row (token, output channel): q = 127 x / max |x| rounded to the nearest (ties to even), scale = max |x| / 127.
//
// The sum is an integer and exact (127^2 K < 2^31 bounds K at 131,072); it becomes f32 (2^-24) before the two scales.  A row whose values
// are not all finite has a scale that is not finite and gives NaN; a row of zeros gives the bias.
// Bound: the integer matrix cores (twice the bf16 rate) for many rows, HBM (the weights once, half the bf16 bytes) for few.
#include "entry_checks.h"
#include "gemm_common.h"
#include <type_traits>

namespace {

inline int ok() { return hipGetLastError() == hipSuccess ? MMSUM_OK : MMSUM_ERR_HIP; }
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef u32x4_t u32x4_a4_t __attribute__((aligned(4)));

// ---- quantisation ------------------------------------------------------------------------------------------------------------------
// 127 x first, so that x = max / 2 lands on the tie it is; the quotient by max correctly rounded: with rc = 1 / max rounded to the nearest,
// q = y rc is within an ulp, y - q max is exact in an fma, and q + (y - q max) rc rounds to the quotient (Markstein).  Rows near either end
// of the f32 range are moved by 2^64 first.  The maximum is taken over the bits of |x|, where NaN is larger than infinity: it survives.
struct RowQuant { float mul, top, rc, scale; bool zero; };
__device__ __forceinline__ RowQuant row_quant(uint32_t top_bits) {
    const float top = __builtin_bit_cast(float, top_bits);
    const float pre = top > 0x1p100f ? 0x1p-64f : top < 0x1p-60f ? 0x1p64f : 1.f;
    RowQuant r;
    r.zero = !(top > 0.f && top < INFINITY);                        // nothing to quantise: zeros (a scale that is not finite makes them NaN)
    r.mul = 127.f * pre;
    r.top = top * pre;
    r.rc = 1.f / r.top;
    r.scale = top / 127.f;
    return r;
}
__device__ __forceinline__ int quantize(float x, const RowQuant& r) {
    const float y = x * r.mul, q = y * r.rc;
    return (int)rintf(fmaf(fmaf(-q, r.top, y), r.rc, q));
}
template <typename T> __device__ __forceinline__ void load_row8(const T* __restrict__ x, int k, int K, float (&f)[8]) {
    if (k + 8 <= K) {
        if constexpr (sizeof(T) == 2) {
            typedef u32x4_t v_t __attribute__((aligned(2)));
            const u32x4_t v = *reinterpret_cast<const v_t*>(x + k);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __builtin_bit_cast(float, e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
        } else {
            const u32x4_t a = *reinterpret_cast<const u32x4_a4_t*>(x + k), b = *reinterpret_cast<const u32x4_a4_t*>(x + k + 4);
            __builtin_memcpy(f, &a, 16);
            __builtin_memcpy(f + 4, &b, 16);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = k + e < K ? to_f32(x[k + e]) : 0.f;
    }
}
__device__ __forceinline__ uint32_t top8(uint32_t top, const float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float v = f[e];
        const uint32_t u = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
        top = u > top ? u : top;
    }
    return top;
}
__device__ __forceinline__ u32x2_t pack8(const float (&f)[8], const RowQuant& r) {
    uint32_t w[2] = {0, 0};
    if (!r.zero)
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e >> 2] |= ((uint32_t)quantize(f[e], r) & 255u) << (8 * (e & 3));
    return u32x2_t{w[0], w[1]};
}
__device__ __forceinline__ uint32_t wave_top(uint32_t t) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t v = __shfl_xor((int)t, o);
        t = v > t ? v : t;
    }
    return t;
}

// A wave a row, eight neighbouring values a lane and step, the row held in registers between the maximum and the rounding (K <= 512 CH).
// Bound: HBM (the row once, a byte out for each value).
template <typename T, int CH>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ x, long ldx, int M, int K, int8_t* __restrict__ q, long ldq, float* __restrict__ scale) {
    const int lane = threadIdx.x & 63;
    const long row = block_index() * 4 + (threadIdx.x >> 6);
    if (row >= M) return;
    float f[CH][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) load_row8(x + row * ldx, (i * 64 + lane) * 8, K, f[i]);
#pragma unroll
    for (int i = 0; i < CH; ++i) top = top8(top, f[i]);
    const RowQuant r = row_quant(wave_top(top));
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int k = (i * 64 + lane) * 8;
        if (k < ldq) *reinterpret_cast<u32x2_t*>(q + row * ldq + k) = pack8(f[i], r);
    }
    if (lane == 0) scale[row] = r.scale;
}
// longer rows: a workgroup a row, read twice
template <typename T>
__global__ __launch_bounds__(256) void quantize_long_kernel(const T* __restrict__ x, long ldx, int M, int K, int8_t* __restrict__ q, long ldq, float* __restrict__ scale) {
    __shared__ uint32_t sh[4];
    const long row = block_index();
    if (row >= M) return;
    const int tid = threadIdx.x;
    uint32_t top = 0;
    for (int k = tid * 8; k < K; k += 2048) {
        float f[8];
        load_row8(x + row * ldx, k, K, f);
        top = top8(top, f);
    }
    top = wave_top(top);
    if ((tid & 63) == 0) sh[tid >> 6] = top;
    __syncthreads();
    const uint32_t a = sh[0] > sh[1] ? sh[0] : sh[1], b = sh[2] > sh[3] ? sh[2] : sh[3];
    const RowQuant r = row_quant(a > b ? a : b);
    for (int k = tid * 8; k < (int)ldq; k += 2048) {
        float f[8];
        load_row8(x + row * ldx, k, K, f);
        *reinterpret_cast<u32x2_t*>(q + row * ldq + k) = pack8(f, r);
    }
    if (tid == 0) scale[row] = r.scale;
}
template <typename T>
int launch_quantize(const void* x, long ldx, int M, int K, void* q, long ldq, float* scale, hipStream_t s) {
    const dim3 grid = grid_of((M + 3L) / 4);
    const T* const xt = static_cast<const T*>(x);
    int8_t* const qt = static_cast<int8_t*>(q);
    if (ldq <= 512) hipLaunchKernelGGL((quantize_kernel<T, 1>), grid, dim3(256), 0, s, xt, ldx, M, K, qt, ldq, scale);
    else if (ldq <= 1024) hipLaunchKernelGGL((quantize_kernel<T, 2>), grid, dim3(256), 0, s, xt, ldx, M, K, qt, ldq, scale);
    else if (ldq <= 2048) hipLaunchKernelGGL((quantize_kernel<T, 4>), grid, dim3(256), 0, s, xt, ldx, M, K, qt, ldq, scale);
    else if (ldq <= 4096) hipLaunchKernelGGL((quantize_kernel<T, 8>), grid, dim3(256), 0, s, xt, ldx, M, K, qt, ldq, scale);
    else hipLaunchKernelGGL((quantize_long_kernel<T>), grid_of(M), dim3(256), 0, s, xt, ldx, M, K, qt, ldq, scale);
    return ok();
}

// GELU, erf form: x Phi(x) = max(x, 0) - |x| Phi(-|x|), and Phi(-a) = e^(-a^2 / 2) R(a) with R(a) = erfcx(a / sqrt 2) / 2, a smooth function that a
// polynomial in t = 1 / (1 + p a) fits with a small RELATIVE error (least maximum on 0 .. 14, by reweighted least squares): no cancellation, and the
// tail keeps its digits.  Infinities give the limits, inf and 0.
// For bf16 results: degree 5, p = 0.35, 2.4e-5 of Phi (half a step of bf16 is 2e-3).  14 instructions, two of them transcendental (20 issue slots):
// the many-row kernels' epilogue is bound by them.  36,864 x 4,096 x 1,024, bf16 results 193 us, f32 results 260 (232 with the form for bf16).
__device__ __forceinline__ float gelu_bf16(float x) {
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(x), 0.35f, 1.f));
    const float e = __builtin_amdgcn_exp2f(x * (x * -0.72134752044f));
    const float r = fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.09778264909982681f, 0.27888500690460205f), 0.010943694971501827f), 0.17298974096775055f), 0.13469082117080688f),
                         0.0002850691962521523f);
    return fmaf(-fminf(fabsf(x), 0x1.fffffep+127f), r * e, fmaxf(x, 0.f));
}
// For f32 results: |x| < 1: Phi(x) = 1/2 + x Q(x^2), Q of degree 5 (7e-10), as digits cancel nowhere else; beyond: degree 7, p = 0.6 (7e-8).  Off by 2.4e-7 of
// the result for |x| < 1, 6e-7 down to -3, 1.5e-6 down to -5 (the exponential's argument, rounded, grows with x^2).
__device__ __forceinline__ float gelu_f32(float x) {
    const float a = fabsf(x), u = x * x;
    const float q = fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, -7.654203727724962e-06f, 0.00011348636326147243f), -0.0011863299878314137f), 0.009973322972655296f),
                                 -0.06649035960435867f), 0.3989422917366028f);
    const float t = __builtin_amdgcn_rcpf(fmaf(a, 0.6f, 1.f));
    const float r = fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.19833126664161682f, 0.6180407404899597f), -0.6681910157203674f), 0.1442471593618393f),
                                 0.12018100917339325f), 0.24333792924880981f), 0.2391035407781601f), 7.250037924677599e-06f);
    const float out = fmaf(-fminf(a, 0x1.fffffep+127f), r * __builtin_amdgcn_exp2f(u * -0.72134752044f), fmaxf(x, 0.f));
    return a < 1.f ? fmaf(u, q, 0.5f * x) : out;
}
template <typename T> __device__ __forceinline__ float gelu_i8(float x) { return sizeof(T) == 2 ? gelu_bf16(x) : gelu_f32(x); }

// ---- product -----------------------------------------------------------------------------------------------------------------------
struct I8Args {
    const int8_t* A; long lda; const float* sa; const int8_t* B; long ldb; const float* sb; const float* bias;
    void* C; long ldc; int M, N, K;
};

// eight neighbouring f32 of an array of n (WHOLE: all inside; else the last one in place of those behind it), there when the function returns:
// a first use inside a predicated store would wait for every store issued before it, one by one
template <bool WHOLE> __device__ __forceinline__ void load_cols(const float* __restrict__ p, int c, int n, float (&f)[8]) {
    if constexpr (WHOLE) {
        const u32x4_t a = *reinterpret_cast<const u32x4_a4_t*>(p + c), b = *reinterpret_cast<const u32x4_a4_t*>(p + c + 4);
        __builtin_memcpy(f, &a, 16);
        __builtin_memcpy(f + 4, &b, 16);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = p[c + k < n ? c + k : n - 1];
    }
}
__device__ __forceinline__ void retire(float (&f)[8]) {
#pragma unroll
    for (int k = 0; k < 8; ++k) asm volatile("" : "+v"(f[k]));
}

// eight results of a row of which n are left (WHOLE: all of them); rows may start at any element
template <typename T, bool WHOLE> __device__ __forceinline__ void store_cols(T* o, int n, const float (&v)[8]) {
    if constexpr (!WHOLE) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < n) o[k] = from_f32<T>(v[k]);
    } else if constexpr (sizeof(T) == 2) {
        typedef bf16x8_t v_t __attribute__((aligned(2)));
        bf16x8_t t;
#pragma unroll
        for (int k = 0; k < 8; ++k) t[k] = (bf16_t)v[k];
        *reinterpret_cast<v_t*>(o) = t;
    } else {
        typedef f32x4_t v_t __attribute__((aligned(4)));
        *reinterpret_cast<v_t*>(o) = f32x4_t{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<v_t*>(o + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
    }
}

// Many rows: 256x256 tiles, four waves of 128x128, one a SIMD, 256 accumulator registers each (every AGPR, pinned there as "+a" operands of
// the MFMAs).  Operands pass through LDS in stages of 128 bytes of k: row r at 128 r, its 16-byte chunk c at c ^ ((r >> 1) & 7), which
// spreads a fragment read (row = lane & 15, chunk = lane >> 4) over all banks; the DMA writes LDS linearly, so the XOR sits on the source
// address of its lanes.  LDS holds three stages of A (streamed) and two of B (weights, in L2): 160 KB.
// The stages of ALL tiles of a workgroup form one stream: while the last two stages of a tile are multiplied, the first two of the next
// one are on their way, and they land under the epilogue, which goes from the accumulators straight to memory and leaves LDS alone.
//   stage s: 64 MFMAs on its first 64 k (fragments X) | reads of its second 64 k (Y) | DMA: A of stage s + 2
//            wait for stage s + 1 (only A of s + 2 may be in flight: vmcnt(8)) ; barrier
//            64 MFMAs on Y | reads of stage s + 1's first 64 k (X) | DMA: B of stage s + 2
// The weights ride as the MFMA's A operand, so that a lane's four results are neighbouring columns; within 32 weight rows LDS row
// 16 j + 4 g + e holds weight row 8 g + 4 j + e, and the two MFMAs of a pair leave a lane eight neighbouring columns: a 16-byte store.
// Measured (MI355X): 8192^3 381 us = 2,890 TOP/s (the library's integer product 2,107); 36,864 x 4,096 x 1,024 184 us, with GELU 234: a
// tile's epilogue is 65,536 values of 6 (26 with GELU, counting the transcendentals' four) issue slots on 256 lanes beside 12 us of main loop.
constexpr int kStageBytes = 256 * 128;
template <typename T, bool GELU>
__global__ __launch_bounds__(256, 1) void gemm_i8_w4_kernel(I8Args p) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    constexpr int B_BASE = 3 * kStageBytes;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int tiles_m = (p.M + 255) / 256, tiles_n = (p.N + 255) / 256, total = tiles_m * tiles_n;
    const int nst = p.K / 128;
    int a_frag0, b_frag0, ydelta, offA, offB;                     // per lane; made anew for every tile (lane_constants), so that the epilogue need not carry them

    const int my_tiles = (total - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;     // >= 1: the grid has no more workgroups than tiles
    const int S = my_tiles * nst;
    // the stage that is requested next: tile pvid, stage pst of it, into LDS stages pa / pb
    int pvid = blockIdx.x, pst = 0, pa = 0, pb = 0;
    const int8_t* baseA = nullptr;
    const int8_t* baseB = nullptr;
    int bytesA = 0, bytesB = 0;                                    // from the tile's first row to the operand's end: rows behind it are not fetched (nor their results stored)
    // A piece is eight rows; piece i of wave w covers rows 32 i + 8 w .., so a lane's offset of piece i is that of piece 0 + 32 i rows.
    auto lane_constants = [&]() {
        int ln;
        asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(ln));
        const int row0 = wave * 8 + (ln >> 3), ch0 = ((ln & 7) ^ ((row0 >> 1) & 7)) * 16;
        offA = row0 * (int)p.lda + ch0;
        offB = ((((row0 >> 2) & 3) << 3) | (((row0 >> 4) & 1) << 2) | (row0 & 3)) * (int)p.ldb + ch0;
        const int r16 = ln & 15, fo = r16 * 128 + ((((ln >> 4) ^ (r16 >> 1)) & 7) << 4);
        a_frag0 = wm * 128 * 128 + fo;
        b_frag0 = B_BASE + wn * 128 * 128 + fo;
        ydelta = (fo ^ 64) - fo;
    };
    auto set_tile = [&](int vid) {
        int tm, tn;
        tile_coords(xcd_remap(vid, total), tiles_m, tiles_n, tm, tn);
        baseA = p.A + (long)tm * 256 * p.lda;
        baseB = p.B + (long)tn * 256 * p.ldb;
        const long ra = (p.M - (long)tm * 256) * p.lda, rb = (p.N - (long)tn * 256) * p.ldb;
        bytesA = (int)(ra < 0x7fffffff ? ra : 0x7fffffff);
        bytesB = (int)(rb < 0x7fffffff ? rb : 0x7fffffff);
    };
#if defined(__HIP_DEVICE_COMPILE__)        // the host pass rejects the buffer-resource builtins inside templates
#define I8_DMA(BASE, BYTES, OFF, LDS)                                                                                               \
    {                                                                                                                               \
        typedef __attribute__((address_space(3))) void* lds_ptr;                                                                    \
        const __amdgpu_buffer_rsrc_t r_ = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(BASE), 0, BYTES, 0x00020000);       \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r_, (lds_ptr)(LDS), 16, OFF, pst * 128, 0, 0);                                     \
    }
#else
#define I8_DMA(BASE, BYTES, OFF, LDS) {}
#endif
#define I8_A(I) I8_DMA(baseA, bytesA, oa + (I) * 32 * (int)p.lda, smem + pa * kStageBytes + ((I) * 4 + wave) * 1024)
#define I8_B(I) I8_DMA(baseB, bytesB, ob + (I) * 32 * (int)p.ldb, smem + B_BASE + pb * kStageBytes + ((I) * 4 + wave) * 1024)
    auto advance = [&]() {
        pa = pa == 2 ? 0 : pa + 1;
        pb ^= 1;
        if (++pst == nst) {
            pst = 0;
            pvid += gridDim.x;
            if (pvid < total) set_tile(pvid);
        }
    };

    Frag aX[4], bX[4], aY[4], bY[4];
    set_tile(pvid);
    lane_constants();
    int oa = offA, ob = offB;
#pragma unroll
    for (int i = 0; i < 8; ++i) I8_A(i)
#pragma unroll
    for (int i = 0; i < 8; ++i) I8_B(i)
    advance();
    if (S > 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) I8_A(i)
#pragma unroll
        for (int i = 0; i < 8; ++i) I8_B(i)
        advance();
        asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
    } else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
#define I8_MMA(FA, FB, I, J)                                                                                                         \
    _Pragma("unroll") for (int q = 0; q < 4; ++q)                                                                                    \
        asm volatile("v_mfma_i32_16x16x64_i8 %0, %2, %1, %0" : "+a"(c[I][J][q]) : "v"(FA[I].c[q >> 1]), "v"(FB[J].c[q & 1]) : "memory");
#define I8_MMA0(FA, FB, I, J)                                                                                                        \
    _Pragma("unroll") for (int q = 0; q < 4; ++q)                                                                                    \
        asm volatile("v_mfma_i32_16x16x64_i8 %0, %2, %1, 0" : "=a"(c[I][J][q]) : "v"(FA[I].c[q >> 1]), "v"(FB[J].c[q & 1]) : "memory");
    // LEFT = stages of the stream behind this one: >= 2 steady state; 1: nothing left to request; 0: the last one
    bool whole = false;                                           // the last tile left by the WHOLE epilogue
    auto stage = [&](i32x4_t (&c)[4][4][4], int abuf, int bbuf, auto left_c, auto first_c) {
        constexpr int LEFT = decltype(left_c)::value;
        constexpr bool FIRST = decltype(first_c)::value;
        const char* As = smem + abuf * kStageBytes + a_frag0;
        const char* Bs = smem + bbuf * kStageBytes + b_frag0;
        int oa = offA, ob = offB;
        asm volatile("s_nop 1" : "+v"(oa), "+v"(ob)::"memory");     // opaque: the pieces' 16 offsets are added up here, not carried in registers
#pragma unroll
        for (int g = 0; g < 16; ++g) {
            if constexpr (FIRST) { I8_MMA0(aX, bX, g >> 2, g & 3) } else { I8_MMA(aX, bX, g >> 2, g & 3) }
            if (g < 8) bY[g >> 1].c[g & 1] = *reinterpret_cast<const u32x4_t*>(Bs + ((g >> 1) * 32 + (g & 1) * 16) * 128 + ydelta);
            else aY[(g - 8) >> 1].c[g & 1] = *reinterpret_cast<const u32x4_t*>(As + (((g - 8) >> 1) * 32 + (g & 1) * 16) * 128 + ydelta);
            if constexpr (LEFT >= 2) { if (!(g & 1)) I8_A(g >> 1) }
        }
        // vmcnt counts down in order: behind stage s + 1's pieces come, in a tile's first stage, the last tile's 32 stores of a whole bf16
        // epilogue (its loads are back before its first store), which may stay in flight (check_handoff.py: the build fails unless they are 32)
        if constexpr (LEFT >= 2 && FIRST && sizeof(T) == 2) {
            if (whole) asm volatile("s_waitcnt vmcnt(40)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        } else if constexpr (LEFT >= 2) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        else if constexpr (LEFT == 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_nop 1" ::: "memory");
        __builtin_amdgcn_s_barrier();
        const char* An = smem + (abuf == 2 ? 0 : abuf + 1) * kStageBytes + a_frag0;
        const char* Bn = smem + (bbuf ^ 1) * kStageBytes + b_frag0;
#pragma unroll
        for (int g = 0; g < 16; ++g) {
            I8_MMA(aY, bY, g >> 2, g & 3)
            if constexpr (LEFT >= 1) {
                if (g < 8) bX[g >> 1].c[g & 1] = *reinterpret_cast<const u32x4_t*>(Bn + ((g >> 1) * 32 + (g & 1) * 16) * 128);
                else aX[(g - 8) >> 1].c[g & 1] = *reinterpret_cast<const u32x4_t*>(An + (((g - 8) >> 1) * 32 + (g & 1) * 16) * 128);
            }
            if constexpr (LEFT >= 2) { if (!(g & 1)) I8_B(g >> 1) }
        }
        if constexpr (LEFT >= 2) advance();
    };
    using std::integral_constant;
    int s = 0, abuf = 0, bbuf = 0;
    for (int vid = blockIdx.x; vid < total; vid += gridDim.x) {
        i32x4_t c[4][4][4];                                       // [32 rows][32 columns][quarter q = 2 (row half) + (column half)]
        lane_constants();
        // (read here and not kept from the last tile's last stage, which would cost the epilogue 64 registers)
#pragma unroll
        for (int g = 0; g < 8; ++g) {
            bX[g >> 1].c[g & 1] = *reinterpret_cast<const u32x4_t*>(smem + bbuf * kStageBytes + b_frag0 + ((g >> 1) * 32 + (g & 1) * 16) * 128);
            aX[g >> 1].c[g & 1] = *reinterpret_cast<const u32x4_t*>(smem + abuf * kStageBytes + a_frag0 + ((g >> 1) * 32 + (g & 1) * 16) * 128);
        }
        auto next = [&]() {
            ++s;
            abuf = abuf == 2 ? 0 : abuf + 1;
            bbuf ^= 1;
        };
        if (s + 2 < S) stage(c, abuf, bbuf, integral_constant<int, 2>{}, std::true_type{});
        else if (s + 2 == S) stage(c, abuf, bbuf, integral_constant<int, 1>{}, std::true_type{});
        else stage(c, abuf, bbuf, integral_constant<int, 0>{}, std::true_type{});
        next();
        const int end = s + nst - 1, full = end < S - 2 ? end : S - 2;
        while (s < full) { stage(c, abuf, bbuf, integral_constant<int, 2>{}, std::false_type{}); next(); }
        if (s < end && s + 2 == S) { stage(c, abuf, bbuf, integral_constant<int, 1>{}, std::false_type{}); next(); }
        if (s < end) { stage(c, abuf, bbuf, integral_constant<int, 0>{}, std::false_type{}); next(); }
        asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");       // the last MFMAs' results: the compiler does not know they are still on their way
        int tm, tn, lane_e;
        tile_coords(xcd_remap(vid, total), tiles_m, tiles_n, tm, tn);
        asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane_e));
        const int mr = tm * 256 + wm * 128 + (lane_e & 15), nc = tn * 256 + wn * 128 + 8 * (lane_e >> 4);
        auto epilogue = [&](auto whole_c) {
            constexpr bool WHOLE = decltype(whole_c)::value;      // every row and column of the tile is stored, in whole chunks
            float sx[8], sw[4][8], bs[4][8] = {};
#pragma unroll
            for (int k = 0; k < 8; ++k) sx[k] = p.sa[WHOLE || mr + 16 * k < p.M ? mr + 16 * k : p.M - 1];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                load_cols<WHOLE>(p.sb, nc + 32 * j, p.N, sw[j]);
                if (p.bias != nullptr) load_cols<WHOLE>(p.bias, nc + 32 * j, p.N, bs[j]);
            }
            retire(sx);
#pragma unroll
            for (int j = 0; j < 4; ++j) { retire(sw[j]); retire(bs[j]); }
            __builtin_amdgcn_sched_barrier(0);
            T* row = static_cast<T*>(p.C) + (long)mr * p.ldc + nc;
#pragma unroll
            for (int k = 0; k < 8; ++k, row += 16 * p.ldc) {
                if (WHOLE || mr + 16 * k < p.M) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            v[e] = fmaf((float)c[k >> 1][j][2 * (k & 1) + (e >> 2)][e & 3] * sx[k], sw[j][e], bs[j][e]);
                            if constexpr (GELU) v[e] = gelu_i8<T>(v[e]);
                        }
                        store_cols<T, WHOLE>(row + 32 * j, p.N - nc - 32 * j, v);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        };
        whole = tm * 256 + 256 <= p.M && tn * 256 + 256 <= p.N;
        if (whole) epilogue(std::true_type{});
        else epilogue(std::false_type{});
    }
#undef I8_MMA0
#undef I8_MMA
#undef I8_B
#undef I8_A
#undef I8_DMA
}

// One tile of BM x BN a workgroup of WM x WN waves, the stages in a ring that runs NST - 1 of them ahead of the products, at most 80 KB of
// LDS: two workgroups a CU, and the main loop of one runs under the waits and the epilogue of the other.  Operand rows, swizzle and the order
// of the weight rows as above.  192x128 (two stages) for large products of a short sum, where the epilogue weighs; 64x64 (four) for small ones.
// Measured (MI355X, 192x128): 36,864 x 4,096 x 1,024 178 us, with GELU 193 - 207 launch after launch (228 in a kernel trace, every launch on an idle
// card); 36,864 x 1,024 x 4,096 127 us = 2,435 TOP/s.  38,400 x 3,584 x 1,024, plain | GELU: matrix cores busy 39 | 36 % of the cycles, vector units 29 | 61 %:
// with GELU the two take turns.
template <typename T, bool GELU, int BM, int BN, int WM, int WN, int NST>
__global__ __launch_bounds__(WM* WN * 64, 2) void gemm_i8_ring_kernel(I8Args p) {
    constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, STAGE = (BM + BN) * 128, PA = BM / 8 / NW, PB = BN / 8 / NW, PPW = PA + PB;
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "whole pieces for every wave");
    static_assert(NST * STAGE <= 81920, "two workgroups a CU");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN;
    int tm, tn;
    tile_coords(xcd_remap(blockIdx.x, gridDim.x), tiles_m, tiles_n, tm, tn);
    const int nst = p.K / 128;
    const long ra = (p.M - (long)tm * BM) * p.lda, rb = (p.N - (long)tn * BN) * p.ldb;
    const int bytesA = (int)(ra < 0x7fffffff ? ra : 0x7fffffff), bytesB = (int)(rb < 0x7fffffff ? rb : 0x7fffffff);
    const int8_t* const baseA = p.A + (long)tm * BM * p.lda;
    const int8_t* const baseB = p.B + (long)tn * BN * p.ldb;
    int offA[PA], offB[PB];                                        // piece i of a wave: rows 8 (NW i + wave) .. + 7
#pragma unroll
    for (int i = 0; i < PA; ++i) {
        const int row = (i * NW + wave) * 8 + (lane >> 3);
        offA[i] = row * (int)p.lda + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
    }
#pragma unroll
    for (int i = 0; i < PB; ++i) {
        const int row = (i * NW + wave) * 8 + (lane >> 3), wrow = (row & ~31) | (((row >> 2) & 3) << 3) | (((row >> 4) & 1) << 2) | (row & 3);
        offB[i] = wrow * (int)p.ldb + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
    }
    auto issue = [&](int st) {
#if defined(__HIP_DEVICE_COMPILE__)
        typedef __attribute__((address_space(3))) void* lds_ptr;
        const __amdgpu_buffer_rsrc_t da = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(baseA), 0, bytesA, 0x00020000);
        const __amdgpu_buffer_rsrc_t db = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(baseB), 0, bytesB, 0x00020000);
        char* const slot = smem + st % NST * STAGE;
#pragma unroll
        for (int i = 0; i < PA; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(da, (lds_ptr)(slot + (i * NW + wave) * 1024), 16, offA[i], st * 128, 0, 0);
#pragma unroll
        for (int i = 0; i < PB; ++i) __builtin_amdgcn_raw_ptr_buffer_load_lds(db, (lds_ptr)(slot + BM * 128 + (i * NW + wave) * 1024), 16, offB[i], st * 128, 0, 0);
#endif
    };
    const int r16 = lane & 15, fo = r16 * 128 + ((((lane >> 4) ^ (r16 >> 1)) & 7) << 4);
    i32x4_t c[TM][TN][4] = {};
#pragma unroll
    for (int st = 0; st < NST - 1; ++st)
        if (st < nst) issue(st);
    for (int st = 0; st < nst; ++st) {
        const int ahead = nst - 1 - st;                            // stages requested behind this one, NST - 2 of them at most
        // (lgkmcnt: this wave's reads of stage st - 1 are back; its slot is requested into behind the barrier)
        if (ahead >= NST - 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * PPW) : "memory");
        else if (NST > 3 && ahead == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(PPW) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");                               // no read of the stage above its barrier
        const char* const A = smem + st % NST * STAGE + wm * (TM * 32) * 128 + fo;
        const char* const B = smem + st % NST * STAGE + BM * 128 + wn * (TN * 32) * 128 + fo;
        const int yd = (fo ^ 64) - fo;
        i32x4_t a[2][TM][2], b[2][TN][2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) a[y][i][h] = *reinterpret_cast<const i32x4_t*>(A + (i * 32 + h * 16) * 128 + y * yd);
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) b[y][j][h] = *reinterpret_cast<const i32x4_t*>(B + (j * 32 + h * 16) * 128 + y * yd);
        }
        if (st + NST - 1 < nst) issue(st + NST - 1);               // into the slot of stage st - 1: every wave is past its products
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) c[i][j][q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[y][j][q & 1], a[y][i][q >> 1], c[i][j][q], 0, 0, 0);
    }
    const int mr = tm * BM + wm * (TM * 32) + r16, nc = tn * BN + wn * (TN * 32) + 8 * (lane >> 4);
    auto epilogue = [&](auto whole_c) {
        constexpr bool WHOLE = decltype(whole_c)::value;
        float sx[2 * TM], sw[TN][8], bs[TN][8] = {};
#pragma unroll
        for (int k = 0; k < 2 * TM; ++k) sx[k] = p.sa[WHOLE || mr + 16 * k < p.M ? mr + 16 * k : p.M - 1];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            load_cols<WHOLE>(p.sb, nc + 32 * j, p.N, sw[j]);
            if (p.bias != nullptr) load_cols<WHOLE>(p.bias, nc + 32 * j, p.N, bs[j]);
        }
#pragma unroll
        for (int k = 0; k < 2 * TM; ++k) asm volatile("" : "+v"(sx[k]));
#pragma unroll
        for (int j = 0; j < TN; ++j) { retire(sw[j]); retire(bs[j]); }
        T* row = static_cast<T*>(p.C) + (long)mr * p.ldc + nc;
#pragma unroll
        for (int k = 0; k < 2 * TM; ++k, row += 16 * p.ldc) {
            if (WHOLE || mr + 16 * k < p.M) {
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[e] = fmaf((float)c[k >> 1][j][2 * (k & 1) + (e >> 2)][e & 3] * sx[k], sw[j][e], bs[j][e]);
                        if constexpr (GELU) v[e] = gelu_i8<T>(v[e]);
                    }
                    store_cols<T, WHOLE>(row + 32 * j, p.N - nc - 32 * j, v);
                }
            }
        }
    };
    if (tm * BM + BM <= p.M && tn * BN + BN <= p.N) epilogue(std::true_type{});
    else epilogue(std::false_type{});
}

// Few rows (a decode step): the weights go past the matrix cores once.  A workgroup owns 16 NB columns, its four waves every fourth 64 bytes
// of k; a wave asks for U steps of weights and activations together, straight into the MFMA's registers, and the four partial sums
// meet in LDS.  Integer sums: the order does not matter.
// FUSED: the workgroup quantises the rows itself, into LDS, first -- cheaper than a launch of its own while rows and workgroups are few.
// Bound: HBM / latency.
template <typename T, bool GELU, int MB, int NB, bool FUSED, typename X>
__global__ __launch_bounds__(256) void gemm_i8_few_kernel(I8Args p, const X* __restrict__ x, long ldx, int Kx) {
    constexpr int U = NB == 1 ? 4 : 2, PITCH = 16 * NB + 4;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int* const part = reinterpret_cast<int*>(smem);                 // [4][16 MB][PITCH]
    float* const rs = reinterpret_cast<float*>(smem + 4 * 16 * MB * PITCH * 4);
    char* const xq = smem + 4 * 16 * MB * PITCH * 4 + 64 * MB;      // FUSED: rows of K + 16 bytes
    const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, kg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const long n0 = (long)blockIdx.x * (16 * NB);
    const int xpitch = p.K + 16;
    const int steps = p.K / 64;
    const int8_t* wrow[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) wrow[j] = p.B + (n0 + 16 * j + r16 < p.N ? n0 + 16 * j + r16 : p.N - 1) * p.ldb + kg * 16;
    i32x4_t b[U][NB];
    auto load_weights = [&](int s0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int st = s0 + 4 * u < steps ? s0 + 4 * u : s0 < steps ? s0 : 0;      // behind the end: any step, not multiplied
#pragma unroll
            for (int j = 0; j < NB; ++j) b[u][j] = *reinterpret_cast<const i32x4_t*>(wrow[j] + (long)st * 64);
        }
    };
    load_weights(wave);                                             // on their way while the rows are quantised
    if constexpr (FUSED) {
        for (int m = wave; m < p.M; m += 4) {
            uint32_t top = 0;
            for (int k = lane * 8; k < Kx; k += 512) {
                float f[8];
                load_row8(x + m * ldx, k, Kx, f);
                top = top8(top, f);
            }
            const RowQuant r = row_quant(wave_top(top));
            for (int k = lane * 8; k < p.K; k += 512) {
                float f[8];
                load_row8(x + m * ldx, k, Kx, f);
                *reinterpret_cast<u32x2_t*>(xq + m * xpitch + k) = pack8(f, r);
            }
            if (lane == 0) rs[m] = r.scale;
        }
        __syncthreads();
    } else if (tid < p.M) rs[tid] = p.sa[tid];
    i32x4_t acc[MB][NB] = {};
    for (int s0 = wave; s0 < steps; s0 += 4 * U) {
        if (s0 != wave) load_weights(s0);
        i32x4_t a[U][MB];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int st = s0 + 4 * u < steps ? s0 + 4 * u : s0;
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const int m = 16 * i + r16 < p.M ? 16 * i + r16 : p.M - 1;
                if constexpr (FUSED) a[u][i] = *reinterpret_cast<const i32x4_t*>(xq + m * xpitch + st * 64 + kg * 16);
                else a[u][i] = *reinterpret_cast<const i32x4_t*>(p.A + m * p.lda + st * 64 + kg * 16);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + 4 * u < steps)
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int j = 0; j < NB; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[u][j], a[u][i], acc[i][j], 0, 0, 0);
    }
    // weights as the A operand: a lane holds columns 4 kg .. + 3 of row r16
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) *reinterpret_cast<i32x4_t*>(part + (wave * 16 * MB + 16 * i + r16) * PITCH + 16 * j + 4 * kg) = acc[i][j];
    __syncthreads();
    for (int o = tid; o < p.M * 16 * NB; o += 256) {
        const int m = o / (16 * NB), c = o % (16 * NB);
        const long n = n0 + c;
        if (n >= p.N) continue;
        int sum = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) sum += part[(w * 16 * MB + m) * PITCH + c];
        float v = fmaf((float)sum * rs[m], p.sb[n], p.bias ? p.bias[n] : 0.f);
        if constexpr (GELU) v = gelu_i8<T>(v);
        static_cast<T*>(p.C)[m * p.ldc + n] = from_f32<T>(v);
    }
}

// CUs of the device, a multiple of 8 (the tile walk hands every XCD its own stretch of the tile list)
int cu_count() {
    int dev = 0, v = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || v < 8) return 256;
    return v & ~7;
}

constexpr long kMaxGroups = 0xffffff;        // workgroups of 256 threads that an axis of a launch holds; products beyond (few rows, 2^29 columns and more) are refused
template <typename T, bool GELU, int MB, int NB, bool FUSED, typename X>
int launch_few(const I8Args& p, const X* x, long ldx, int Kx, hipStream_t s) {
    const long blocks = (p.N + 16L * NB - 1) / (16 * NB);
    if (blocks > kMaxGroups) return MMSUM_ERR_BAD_SHAPE;
    const size_t lds = 4 * 16 * MB * (16 * NB + 4) * 4 + 64 * MB + (FUSED ? (size_t)p.M * (p.K + 16) : 0);
    if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_i8_few_kernel<T, GELU, MB, NB, FUSED, X>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
        return MMSUM_ERR_HIP;
    hipLaunchKernelGGL((gemm_i8_few_kernel<T, GELU, MB, NB, FUSED, X>), dim3((unsigned)blocks), dim3(256), lds, s, p, x, ldx, Kx);
    return ok();
}

template <typename T, bool GELU, int BM, int BN, int WM, int WN, int NST>
int launch_ring(const I8Args& p, hipStream_t s) {
    const long tiles = (p.M + (long)BM - 1) / BM * ((p.N + (long)BN - 1) / BN);
    if (tiles > kMaxGroups) return MMSUM_ERR_BAD_SHAPE;
    const size_t lds = (size_t)NST * (BM + BN) * 128;
    if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_i8_ring_kernel<T, GELU, BM, BN, WM, WN, NST>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess)
        return MMSUM_ERR_HIP;
    hipLaunchKernelGGL((gemm_i8_ring_kernel<T, GELU, BM, BN, WM, WN, NST>), dim3((unsigned)tiles), dim3(WM * WN * 64), lds, s, p);
    return ok();
}

// The kernel of a product: family, tile (few rows: rows and columns of a workgroup), workgroups
struct I8Plan { int kernel, bm, bn; long groups; };
I8Plan plan_product(int M, int N, int K, bool gelu) {
    auto up = [](long a, long b) { return (a + b - 1) / b; };
    if (M <= 64) {
        // Workgroups of 64 columns read the activations less often, of 16 columns fill more CUs (us, 16 | 64 columns, K = 1,024): N = 8,192: 1 row 3.4 | 4.2,
        // 32 rows 4.9 | 5.9; 16,384: 1 row 4.3 | 5.0, 16 rows 5.5 | 5.7, 32 rows 7.8 | 6.1; 50,265: 1 row 10.8 | 10.8, 32 rows 21.5 | 15.9
        const int bn = N >= (M <= 16 ? 32768 : 16384) ? 64 : 16;
        return {MMSUM_I8_PLAN_FEW, M <= 16 ? 16 : M <= 32 ? 32 : 64, bn, up(N, bn)};
    }
    // The tile whose rounds of the CUs take the least time, in tenths of a us: so much a stage of 128 k and so much an epilogue, fitted to the
    // three on 24 shapes (worst choice 9 % over the best).  Measured (us, 64x64 | 192x128 | 256x256, bf16 out):
    //   36,864 x 4,096 x 1,024   318 | 178 | 184, with GELU 345 | 207 | 234        8,192 x 8,192 x 8,192    778 | 445 | 381
    //   36,864 x 1,024 x 4,096   223 | 127 | 141 (2 1/4 rounds of 256x256)        16,384 x 4,096 x 4,096   400 | 237 | 205 (5 3/8 of 192x128)
    //    9,216 x 1,024 x 1,024    23 |  16 |  20                                    2,048 x 2,048 x 2,048    16 |  23 |  19
    //   256 x 50,265 x 1,024      36 |  37 |  27                                      128 x 50,265 x 1,024    21 |  27 |  22
    // The larger tiles are not for fewer than 129 rows: their loads of the missing rows still take their turn.
    const long cus = cu_count(), st = K / 128;
    const long t256 = up(M, 256) * up(N, 256), t192 = up(M, 192) * up(N, 128), t64 = up(M, 64) * up(N, 64);
    const long half = up(t192, cus);                               // rounds of one workgroup a CU: two at once take 4/3 of one alone
    const long us256 = up(t256, cus) * (14 * st + 70 + (gelu ? 50 : 0)), us192 = (2 * half + half % 2) * (11 * st + 60 + (gelu ? 20 : 0)) / 4, us64 = up(t64, 2 * cus) * (4 * st + 14);
    if (M <= 128 || (us64 <= us192 && us64 <= us256)) return {MMSUM_I8_PLAN_RING, 64, 64, t64};
    if (us192 <= us256) return {MMSUM_I8_PLAN_RING, 192, 128, t192};
    return {MMSUM_I8_PLAN_W4, 256, 256, t256 < cus ? t256 : cus};
}

template <typename T, bool GELU>
int launch_product(const I8Args& p, hipStream_t s) {
    const I8Plan g = plan_product(p.M, p.N, p.K, GELU);
    if (g.kernel == MMSUM_I8_PLAN_FEW) {
        if (g.bm == 16) return g.bn == 64 ? launch_few<T, GELU, 1, 4, false, float>(p, nullptr, 0, 0, s) : launch_few<T, GELU, 1, 1, false, float>(p, nullptr, 0, 0, s);
        if (g.bm == 32) return g.bn == 64 ? launch_few<T, GELU, 2, 4, false, float>(p, nullptr, 0, 0, s) : launch_few<T, GELU, 2, 1, false, float>(p, nullptr, 0, 0, s);
        return g.bn == 64 ? launch_few<T, GELU, 4, 4, false, float>(p, nullptr, 0, 0, s) : launch_few<T, GELU, 4, 1, false, float>(p, nullptr, 0, 0, s);
    }
    if ((p.M + 63L) / 64 * ((p.N + 63L) / 64) > 0x7fffffffL) return MMSUM_ERR_BAD_SHAPE;
    if (g.bm == 64) return launch_ring<T, GELU, 64, 64, 2, 2, 4>(p, s);
    if (g.bm == 192) return launch_ring<T, GELU, 192, 128, 2, 2, 2>(p, s);
    const size_t lds = 5 * kStageBytes;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(gemm_i8_w4_kernel<T, GELU>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) return MMSUM_ERR_HIP;
    hipLaunchKernelGGL((gemm_i8_w4_kernel<T, GELU>), dim3((unsigned)g.groups), dim3(256), lds, s, p);
    return ok();
}

// Quantisation and product.  In one launch for up to 8,192 values: there every workgroup's quantising all rows costs no more than the launch (us,
// two | one, N = 1,024): 1 x 1,024 4.8 | 3.5, 1 x 4,096 9.2 | 7.6, 8 x 1,024 5.2 | 5.0, 16 x 1,024 5.4 | 7.7, 8 x 4,096 10.0 | 12.9; 8 x 1,024 into 16,384
// columns 7.4 | 7.8, into 50,265 15.9 | 19.4.
bool quantises_inside(int M, int N, int K) { return M <= 16 && (long)M * K <= 8192 && N <= 16384; }
template <typename T, bool GELU>
int launch_linear(int dtype, const void* x, long ldx, I8Args p, int Kx, hipStream_t s) {
    if (quantises_inside(p.M, p.N, p.K)) {
        if (dtype == MMSUM_BF16) return launch_few<T, GELU, 1, 1, true, bf16_t>(p, static_cast<const bf16_t*>(x), ldx, Kx, s);
        return launch_few<T, GELU, 1, 1, true, float>(p, static_cast<const float*>(x), ldx, Kx, s);
    }
    int8_t* const q = const_cast<int8_t*>(p.A);
    float* const scale = const_cast<float*>(p.sa);
    const int rc = dtype == MMSUM_BF16 ? launch_quantize<bf16_t>(x, ldx, p.M, Kx, q, p.K, scale, s) : launch_quantize<float>(x, ldx, p.M, Kx, q, p.K, scale, s);
    return rc == MMSUM_OK ? launch_product<T, GELU>(p, s) : rc;
}

}  // namespace

extern "C" int mmsum_quantize_i8(int dtype, const void* x, long ldx, int M, int K, void* q, long ldq, float* scale, void* stream) {
    if (M <= 0 || K <= 0 || ldx < K || ldq < K || ldq % 128 || ldq > 0x7fffffc0L) return MMSUM_ERR_BAD_SHAPE;
    if (dtype != MMSUM_BF16 && dtype != MMSUM_F32) return MMSUM_ERR_BAD_DTYPE;
    if (any_null(x, q, scale) || ((uintptr_t)q & 15) || ((uintptr_t)x & (dtype == MMSUM_BF16 ? 1 : 3))) return MMSUM_ERR_BAD_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MMSUM_BF16) return launch_quantize<bf16_t>(x, ldx, M, K, q, ldq, scale, s);
    return launch_quantize<float>(x, ldx, M, K, q, ldq, scale, s);
}

extern "C" int mmsum_gemm_i8(const void* qx, long ldx, const float* sx, const void* qw, long ldw, const float* sw, const float* bias, int dtype_out, void* y, long ldy,
                             int M, int N, int K, int gelu, void* stream) {
    if (M <= 0 || N <= 0 || K <= 0 || K % 128 || K > 131072 || ldx < K || ldw < K || ldx % 16 || ldw % 16 || ldx > 0x3fffff || ldw > 0x3fffff || ldy < N) return MMSUM_ERR_BAD_SHAPE;
    if (dtype_out != MMSUM_BF16 && dtype_out != MMSUM_F32) return MMSUM_ERR_BAD_DTYPE;
    if (any_null(qx, sx, qw, sw, y) || (((uintptr_t)qx | (uintptr_t)qw) & 15) || ((uintptr_t)y & (dtype_out == MMSUM_BF16 ? 1 : 3))) return MMSUM_ERR_BAD_ALIGN;
    I8Args p = {static_cast<const int8_t*>(qx), ldx, sx, static_cast<const int8_t*>(qw), ldw, sw, bias, y, ldy, M, N, K};
    hipStream_t s = (hipStream_t)stream;
    if (dtype_out == MMSUM_BF16) return gelu ? launch_product<bf16_t, true>(p, s) : launch_product<bf16_t, false>(p, s);
    return gelu ? launch_product<float, true>(p, s) : launch_product<float, false>(p, s);
}

extern "C" long mmsum_linear_i8_workspace(int M, int K) { return M <= 0 || K <= 0 || K > 131072 ? 0 : M * ((K + 127L) / 128 * 128 + 4L); }
extern "C" int mmsum_linear_i8(int dtype, const void* x, long ldx, const void* qw, long ldw, const float* sw, const float* bias, int dtype_out, void* y, long ldy, int M,
                               int N, int K, int gelu, void* workspace, void* stream) {
    if (M <= 0 || N <= 0 || K <= 0 || K > 131072 || ldx < K || ldw < (K + 127L) / 128 * 128 || ldw % 16 || ldw > 0x3fffff || ldy < N) return MMSUM_ERR_BAD_SHAPE;
    if ((dtype != MMSUM_BF16 && dtype != MMSUM_F32) || (dtype_out != MMSUM_BF16 && dtype_out != MMSUM_F32)) return MMSUM_ERR_BAD_DTYPE;
    if (workspace == nullptr) return MMSUM_ERR_WORKSPACE;
    if (any_null(x, qw, sw, y) || ((uintptr_t)x & (dtype == MMSUM_BF16 ? 1 : 3)) || (((uintptr_t)qw | (uintptr_t)workspace) & 15) || ((uintptr_t)y & (dtype_out == MMSUM_BF16 ? 1 : 3)))
        return MMSUM_ERR_BAD_ALIGN;
    const int Kp = (K + 127) / 128 * 128;
    int8_t* const q = static_cast<int8_t*>(workspace);
    const float* const scale = reinterpret_cast<const float*>(q + (long)M * Kp);
    I8Args p = {q, Kp, scale, static_cast<const int8_t*>(qw), ldw, sw, bias, y, ldy, M, N, Kp};
    hipStream_t s = (hipStream_t)stream;
    if (dtype_out == MMSUM_BF16) return gelu ? launch_linear<bf16_t, true>(dtype, x, ldx, p, K, s) : launch_linear<bf16_t, false>(dtype, x, ldx, p, K, s);
    return gelu ? launch_linear<float, true>(dtype, x, ldx, p, K, s) : launch_linear<float, false>(dtype, x, ldx, p, K, s);
}

extern "C" int mmsum_linear_i8_plan(int M, int N, int K, int gelu, int quantise, int* plan) {
    if (M <= 0 || N <= 0 || K <= 0 || K > 131072 || (!quantise && K % 128)) return MMSUM_ERR_BAD_SHAPE;
    if (plan == nullptr) return MMSUM_ERR_BAD_ALIGN;
    const int Kp = (K + 127) / 128 * 128;
    const I8Plan g = quantise && quantises_inside(M, N, Kp) ? I8Plan{MMSUM_I8_PLAN_FEW_QUANTISING, 16, 16, (N + 15L) / 16} : plan_product(M, N, Kp, gelu != 0);
    if (g.groups > 0x7fffffffL) return MMSUM_ERR_BAD_SHAPE;
    plan[0] = g.kernel; plan[1] = g.bm; plan[2] = g.bn; plan[3] = (int)g.groups;
    return MMSUM_OK;
}
