// Losses on the log-probabilities of given tokens: scoring, the paired preference loss, the clipped policy loss with a KL term.
//
// A row is one position's V logits x, y its label; m = max x, s = sum exp(x - m):
//   log p(y) = (x_y - m) - log s          d log p(y) / d x_v = [v == y] - exp(x_v - m) / s
// so every loss here is a number c = dL / d log p(y) per row, and its gradient is c ([v == y] - exp(x_v - m) / s).  A label outside
// 0 .. V-1 marks a position that does not count: log p = 0, c = 0, a row of zeros, and its logits are not read.
//
// Bound: HBM.  The policy loss knows c as soon as the row's own log p is known, so its kernel reads the logits once and writes the
// gradient once, the row waiting in registers in between.  The preference loss needs the sums over both summaries of a pair first:
// statistics (read), the pairs' sums and factors, gradient (read, write).
// Measured (MI355X, 50,265 bf16 logits, whole calls one after the other): scoring 72 x 141 rows 177 us (4.7 TB/s), policy loss 72 x 128 rows 317 us (5.3
// TB/s), preference loss of 36 pairs x 128 rows 425 us (4.0 TB/s of what has to move, 5.8 with the second reading); the results' memory new or reused
// alike.  In a kernel trace, where every launch finds the card idle, the policy kernel takes 313 - 388 us, 358 in the middle.
// A row is summed in f32, sequences and means in 64 bits, in an order that depends on the sizes alone.
#include "entry_checks.h"
#include "mmsum_device.h"
#include "mmsum_kernels.h"

namespace {

inline int ok() { return hipGetLastError() == hipSuccess ? MMSUM_OK : MMSUM_ERR_HIP; }

// 16 bytes of a row that starts at any element: packed [N, T, V] logits with an odd V have rows at odd multiples of the element size
template <typename T> struct Chunk;
template <> struct Chunk<bf16_t> { typedef u32x4_t type __attribute__((aligned(2))); };
template <> struct Chunk<float> { typedef u32x4_t type __attribute__((aligned(4))); };
template <typename T> constexpr int kPer = 16 / (int)sizeof(T);

// columns [c, c + kPer) of a row, -inf behind V (adds nothing to a maximum or a sum of exponentials); LAST: read past the caches
template <typename T, bool LAST = false> __device__ __forceinline__ u32x4_t load_chunk(const T* x, int c, int V) {
    if (c + kPer<T> <= V) {
        if constexpr (LAST) return __builtin_nontemporal_load(reinterpret_cast<const typename Chunk<T>::type*>(x + c));
        else return *reinterpret_cast<const typename Chunk<T>::type*>(x + c);
    }
    T t[kPer<T>];
#pragma unroll
    for (int k = 0; k < kPer<T>; ++k) t[k] = c + k < V ? x[c + k] : from_f32<T>(-INFINITY);
    u32x4_t r;
    __builtin_memcpy(&r, t, 16);
    return r;
}
template <typename T> __device__ __forceinline__ void unpack(const u32x4_t& r, float (&f)[kPer<T>]) {
    T t[kPer<T>];
    __builtin_memcpy(t, &r, 16);
#pragma unroll
    for (int k = 0; k < kPer<T>; ++k) f[k] = to_f32(t[k]);
}
// past the caches: a gradient of the logits' size would push out what the second reading finds there (477 -> 430 us)
template <typename T> __device__ __forceinline__ void store_chunk(T* d, int c, int V, const float (&g)[kPer<T>]) {
    T t[kPer<T>];
#pragma unroll
    for (int k = 0; k < kPer<T>; ++k) t[k] = from_f32<T>(g[k]);
    if (c + kPer<T> <= V) {
        u32x4_t r;
        __builtin_memcpy(&r, t, 16);
        __builtin_nontemporal_store(r, reinterpret_cast<typename Chunk<T>::type*>(d + c));
    } else {
#pragma unroll
        for (int k = 0; k < kPer<T>; ++k)
            if (c + k < V) d[c + k] = t[k];
    }
}
// For the sums, whose log-probabilities are f32 whatever the rows' type.  The hardware's exponential is of base 2, and f32(log2 e) is 1.3e-8 of it too
// small: alone it makes every term of a row too large, 5.8e-8 of the sum on average at 50,265 logits, an error that does not average out over
// tokens.  Its rest as a second constant leaves 1e-9, for one more instruction under the loads (72 x 141 rows 177 us with and without).  f32 rows take
// the library's expf (2e-9).
template <typename T> __device__ __forceinline__ float row_exp(float d) {
    if constexpr (sizeof(T) == 4) return expf(d);
    else return __builtin_amdgcn_exp2f(fmaf(d, 0x1.715476p+0f, d * 0x1.4ae0c0p-26f));
}
// for the gradient: bf16 results keep 8 bits, the shorter form (2^-22) is exact enough
template <typename T> __device__ __forceinline__ float grad_exp(float d) { return sizeof(T) == 2 ? __expf(d) : expf(d); }

template <int NT> __device__ __forceinline__ float block_max(float v, float* sh) {
    v = warp_max(v);
    if constexpr (NT == 64) return v;
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v = fmaxf(v, sh[w]);
    return v;
}
template <int NT> __device__ __forceinline__ float block_sum(float v, float* sh) {
    v = warp_sum(v);
    if constexpr (NT == 64) return v;
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v += sh[w];
    return v;
}

// What the policy loss takes per token besides the logits
struct PolicyArgs {
    const float* old_logp; const float* ref_logp; const float* adv;
    const int64_t* labels; int V;
    const int* counts;              // counted tokens: of kCountParts stretches of the batch (token mean) or of every sequence (sequence mean); NULL: counted here
    int adv_per_token, seq_mean, N, T;
    float lo, hi, kl_coef;
    float* terms;                   // [3][R]: weighted loss, KL estimate, clipped indicator of every row
};
constexpr int kCountParts = 64;

// 1 / (the tokens the mean is over); whole waves come here together, a wave's rows are of one sequence or `row` is the lane's own with counts
__device__ __forceinline__ float policy_weight(const PolicyArgs& p, int row, int lane) {
    const int seq = row / p.T;
    int n = 0;
    if (p.counts == nullptr) {
        const long lo = p.seq_mean ? (long)seq * p.T : 0, hi = p.seq_mean ? lo + p.T : (long)p.N * p.T;
        for (long i = lo + lane; i < hi; i += 64) { const int64_t y = p.labels[i]; n += y >= 0 && y < p.V; }
    } else if (p.seq_mean) {
        return 1.f / (fmaxf((float)p.counts[seq], 1.f) * (float)p.N);
    } else n = p.counts[lane];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
    return 1.f / (fmaxf((float)n, 1.f) * (p.seq_mean ? (float)p.N : 1.f));
}
// e^g - 1 - g, g^2 / 2 near 0: by its series there (to g^9 at 1/2, 2e-9), where the difference has no digits left
__device__ __forceinline__ float exp_rest(float g, float expm1_g) {
    const float s = fmaf(g, fmaf(g, fmaf(g, fmaf(g, fmaf(g, fmaf(g, fmaf(g, 1.f / 362880, 1.f / 40320), 1.f / 5040), 1.f / 720), 1.f / 120), 1.f / 24), 1.f / 6), 0.5f);
    return fabsf(g) < 0.5f ? g * g * s : expm1_g - g;
}
// loss = max(-A r, -A clip(r, lo, hi)) + kl (e^d - d - 1) with r = exp(log p - old), d = ref - log p; returns dL / d log p.
// The bounded branch carries no gradient; the KL estimate (non-negative, unbiased under the sampling policy) gives 1 - e^d.
__device__ __forceinline__ float policy_token(const PolicyArgs& p, int row, float lp, float w, float (&t)[3]) {
    const float ratio = expf(lp - p.old_logp[row]);
    const float a = p.adv[p.adv_per_token ? row : row / p.T];
    const float l1 = -a * ratio, l2 = -a * fminf(fmaxf(ratio, p.lo), p.hi);
    float loss = l1 >= l2 ? l1 : l2, d = l1 >= l2 ? l1 : 0.f, kl = 0.f;
    if (l1 != l1 || l2 != l2) loss = d = l1 + l2;                        // NaN in, NaN out: a comparison would lose it
    if (p.ref_logp != nullptr) {
        const float g = p.ref_logp[row] - lp, e1 = expm1f(g);
        kl = exp_rest(g, e1);
        if (p.kl_coef != 0.f) {                                          // else only reported: an estimate past f32 stays out of the loss
            loss += p.kl_coef * kl;
            d -= p.kl_coef * e1;
        }
    }
    t[0] = w * loss;
    t[1] = w * kl;
    t[2] = l1 < l2 ? w : 0.f;
    return w * d;
}

template <typename T> struct RowArgs {
    const T* logits; long ld; const int64_t* labels; int R, V;
    float* logp; float* stats;      // stats [R][2] = {m, s}; may be NULL
    T* dlogits; long ldd; int W;
    int past;                       // rows below it are read past the caches
    PolicyArgs pol;
};

template <typename T, int NT> __device__ __forceinline__ void zero_cols(T* d, int lo, int hi) {
    for (int c = lo + (int)threadIdx.x; c < hi; c += NT) d[c] = from_f32<T>(0.f);
}

// between two sweeps: the compiler may not carry the unpacked values over
template <int MAXC> __device__ __forceinline__ void keep_packed(u32x4_t (&reg)[MAXC]) {
#pragma unroll
    for (int i = 0; i < MAXC; ++i) asm volatile("" : "+v"(reg[i]));
}

// One workgroup a row, the row in MAXC 16-byte chunks per thread: requested together, kept as loaded (packed), swept for the maximum,
// for the sum and, for the policy loss, for the gradient.
template <typename T, int NT, int MAXC, bool POLICY>
__global__ __launch_bounds__(NT, NT == 512 && !POLICY ? 6 : 4) void row_kernel(RowArgs<T> a) {
    __shared__ float sh[2][NT / 64];
    if (block_index() >= a.R) return;
    const int tid = threadIdx.x, row = (int)block_index();
    const int64_t y = a.labels[row];
    T* const d = POLICY ? a.dlogits + (long)row * a.ldd : nullptr;
    if (y < 0 || y >= a.V) {
        if (tid == 0) {
            a.logp[row] = 0.f;
            if (a.stats) { a.stats[2 * (long)row] = 0.f; a.stats[2 * (long)row + 1] = 1.f; }
            if constexpr (POLICY) {
                const long R = (long)a.pol.N * a.pol.T;
                a.pol.terms[row] = a.pol.terms[R + row] = a.pol.terms[2 * R + row] = 0.f;
            }
        }
        if constexpr (POLICY) {
            const float z[kPer<T>] = {};
            for (int c = tid * kPer<T>; c < a.W; c += NT * kPer<T>) store_chunk(d, c, a.W, z);
        }
        return;
    }
    const T* x = a.logits + (long)row * a.ld;                       // no __restrict__: d may be x
    u32x4_t reg[MAXC];
    if (POLICY || row < a.past) {
#pragma unroll
        for (int i = 0; i < MAXC; ++i) reg[i] = load_chunk<T, true>(x, (i * NT + tid) * kPer<T>, a.V);
    } else {
#pragma unroll
        for (int i = 0; i < MAXC; ++i) reg[i] = load_chunk<T>(x, (i * NT + tid) * kPer<T>, a.V);
    }
    const float xy = to_f32(x[y]);                                   // read before any thread writes: d may be x
    float w = 0.f;
    if constexpr (POLICY) w = policy_weight(a.pol, row, tid & 63);
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < MAXC; ++i) {
        float f[kPer<T>];
        unpack<T>(reg[i], f);
#pragma unroll
        for (int k = 0; k < kPer<T>; ++k) m = fmaxf(m, f[k]);
        __builtin_amdgcn_sched_barrier(0);
    }
    keep_packed(reg);
    m = block_max<NT>(m, sh[0]);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < MAXC; ++i) {
        float f[kPer<T>], part = 0.f;
        unpack<T>(reg[i], f);
#pragma unroll
        for (int k = 0; k < kPer<T>; ++k) part += row_exp<T>(f[k] - m);
        s += part;
        __builtin_amdgcn_sched_barrier(0);
    }
    keep_packed(reg);
    s = block_sum<NT>(s, sh[1]);
    const float lp = (xy - m) - logf(s);
    if (tid == 0) {
        a.logp[row] = lp;
        if (a.stats) { a.stats[2 * (long)row] = m; a.stats[2 * (long)row + 1] = s; }
    }
    if constexpr (POLICY) {
        float t[3];
        const float c0 = policy_token(a.pol, row, lp, w, t);
        if (tid == 0) {
            const long R = (long)a.pol.N * a.pol.T;
            a.pol.terms[row] = t[0];
            a.pol.terms[R + row] = t[1];
            a.pol.terms[2 * R + row] = t[2];
        }
        const float cs = -c0 / s;
#pragma unroll
        for (int i = 0; i < MAXC; ++i) {
            const int c = (i * NT + tid) * kPer<T>;
            if (c < a.V) {
                float f[kPer<T>];
                unpack<T>(reg[i], f);
#pragma unroll
                for (int k = 0; k < kPer<T>; ++k) f[k] = c0 == 0.f ? 0.f : cs * grad_exp<T>(f[k] - m);
                if (y >= c && y < c + kPer<T>) {
#pragma unroll
                    for (int k = 0; k < kPer<T>; ++k)
                        if (c + k == y) f[k] += c0;
                }
                store_chunk(d, c, a.V, f);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        zero_cols<T, NT>(d, a.V, a.W);
    }
}

// The same for rows that do not fit the registers of a workgroup: a running maximum and sum, then the row again for the gradient.
template <typename T, bool POLICY>
__global__ __launch_bounds__(1024) void long_row_kernel(RowArgs<T> a) {
    constexpr int NT = 1024;
    __shared__ float sh[2][NT / 64];
    if (block_index() >= a.R) return;
    const int tid = threadIdx.x, row = (int)block_index();
    const int64_t y = a.labels[row];
    T* const d = POLICY ? a.dlogits + (long)row * a.ldd : nullptr;
    const long R = (long)a.pol.N * a.pol.T;
    if (y < 0 || y >= a.V) {
        if (tid == 0) {
            a.logp[row] = 0.f;
            if (a.stats) { a.stats[2 * (long)row] = 0.f; a.stats[2 * (long)row + 1] = 1.f; }
            if constexpr (POLICY) a.pol.terms[row] = a.pol.terms[R + row] = a.pol.terms[2 * R + row] = 0.f;
        }
        if constexpr (POLICY) zero_cols<T, NT>(d, 0, a.W);
        return;
    }
    const T* x = a.logits + (long)row * a.ld;
    const float xy = to_f32(x[y]);
    float w = 0.f;
    if constexpr (POLICY) w = policy_weight(a.pol, row, tid & 63);
    float m = -INFINITY, s = 0.f;
    for (long c = (long)tid * kPer<T>; c < a.V; c += NT * kPer<T>) {
        float f[kPer<T>], mc = -INFINITY;
        unpack<T>(load_chunk(x, (int)c, a.V), f);
#pragma unroll
        for (int k = 0; k < kPer<T>; ++k) mc = fmaxf(mc, f[k]);
        if (mc > m) { s *= row_exp<T>(m - mc); m = mc; }
        float part = 0.f;
#pragma unroll
        for (int k = 0; k < kPer<T>; ++k) part += f[k] == -INFINITY ? 0.f : row_exp<T>(f[k] - m);      // a thread may see nothing but -inf
        s += part;
    }
    const float mine = m;
    m = block_max<NT>(m, sh[0]);
    s = block_sum<NT>((mine == -INFINITY && s == 0.f) ? 0.f : s * row_exp<T>(mine - m), sh[1]);
    const float lp = (xy - m) - logf(s);
    if (tid == 0) {
        a.logp[row] = lp;
        if (a.stats) { a.stats[2 * (long)row] = m; a.stats[2 * (long)row + 1] = s; }
    }
    if constexpr (POLICY) {
        float t[3];
        const float c0 = policy_token(a.pol, row, lp, w, t);
        if (tid == 0) { a.pol.terms[row] = t[0]; a.pol.terms[R + row] = t[1]; a.pol.terms[2 * R + row] = t[2]; }
        const float cs = -c0 / s;
        for (long c = (long)tid * kPer<T>; c < a.V; c += NT * kPer<T>) {
            float f[kPer<T>];
            unpack<T>(load_chunk(x, (int)c, a.V), f);
#pragma unroll
            for (int k = 0; k < kPer<T>; ++k) f[k] = (c0 == 0.f ? 0.f : cs * grad_exp<T>(f[k] - m)) + (c + k == y ? c0 : 0.f);
            store_chunk(d, (int)c, a.V, f);
        }
        zero_cols<T, NT>(d, a.V, a.W);
    }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// Sum of a sequence's counted log-probabilities; one wave a sequence, lanes stride over its tokens.  In 64 bits: a margin is the difference of
// sums of hundreds, whose steps in f32 (2^-16 at 256) are larger than what the tokens' own rounding leaves of it.
__device__ __forceinline__ void sequence_sum(const float* __restrict__ logp, const int64_t* __restrict__ labels, int n, int T, int V, int lane, double& sum, int& cnt) {
    sum = 0.0;
    cnt = 0;
    for (int t = lane; t < T; t += 64) {
        const int64_t y = labels[(long)n * T + t];
        if (y >= 0 && y < V) { sum += logp[(long)n * T + t]; ++cnt; }
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) cnt += __shfl_xor(cnt, o);
}
__global__ __launch_bounds__(256) void sequence_sum_kernel(const float* logp, const int64_t* labels, int N, int T, int V, int average, float* out) {
    const long nl = block_index() * 4 + (threadIdx.x >> 6);
    if (nl >= N) return;
    const int n = (int)nl, lane = threadIdx.x & 63;
    double s;
    int cnt;
    sequence_sum(logp, labels, n, T, V, lane, s, cnt);
    if (lane == 0) out[n] = (float)(average && cnt > 1 ? s / cnt : s);
}

// log(1 + e^x) without overflow
__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

// Pair i = sequences (i, P + i): h = beta ((S_i - ref_i) - (S_{P+i} - ref_{P+i})), loss_i = (1 - e) softplus(-h) + e softplus(h),
// d loss_i / d h = e - sigmoid(-h).  coef[n] = d (mean loss) / d log p of every counted token of sequence n.
// loss (may be NULL): the mean over the pairs, written by a single workgroup of 16 waves that takes them in turn; else pair_loss is left for a mean.
struct PairArgs {
    const float* logp; const int64_t* labels; const float* ref;
    int P, T, V, average;
    float beta, smoothing;
    float* seq; float* margins; float* pair_loss; float* coef; float* loss;
};
struct PairTerms { float sc, sr, h, dc, dr; };
__device__ __forceinline__ PairTerms pair_terms(const PairArgs& a, int p, int lane) {
    PairTerms t;
    int nc, nr;
    double sc, sr;
    sequence_sum(a.logp, a.labels, p, a.T, a.V, lane, sc, nc);
    sequence_sum(a.logp, a.labels, a.P + p, a.T, a.V, lane, sr, nr);
    if (a.average) {
        sc /= nc > 1 ? nc : 1;
        sr /= nr > 1 ? nr : 1;
    }
    const float ic = a.average ? 1.f / fmaxf((float)nc, 1.f) : 1.f, ir = a.average ? 1.f / fmaxf((float)nr, 1.f) : 1.f;
    t.sc = (float)sc;
    t.sr = (float)sr;
    t.h = (float)((double)a.beta * ((sc - (a.ref ? a.ref[p] : 0.f)) - (sr - (a.ref ? a.ref[a.P + p] : 0.f))));
    const float dh = (a.smoothing - 1.f / (1.f + expf(t.h))) * a.beta / (float)a.P;
    t.dc = dh * ic;
    t.dr = -dh * ir;
    return t;
}
__device__ __forceinline__ float pair_loss_of(const PairArgs& a, float h) {
    return a.smoothing == 0.f ? softplus(-h) : (1.f - a.smoothing) * softplus(-h) + a.smoothing * softplus(h);
}
__global__ __launch_bounds__(1024) void pair_kernel(PairArgs a) {
    __shared__ double sh[16];
    const int lane = threadIdx.x & 63, waves = blockDim.x / 64;
    double mean = 0.0;
    for (long pl = block_index() * waves + (threadIdx.x >> 6); pl < a.P; pl += (long)gridDim.x * gridDim.y * waves) {
        const int p = (int)pl;
        const PairTerms t = pair_terms(a, p, lane);
        const float l = pair_loss_of(a, t.h);
        mean += l;
        if (lane == 0) {
            a.seq[p] = t.sc;
            a.seq[a.P + p] = t.sr;
            a.margins[p] = t.h;
            a.pair_loss[p] = l;
            a.coef[p] = t.dc;
            a.coef[a.P + p] = t.dr;
        }
    }
    if (a.loss != nullptr) {                                       // one workgroup of 16 waves
        if (lane == 0) sh[threadIdx.x >> 6] = mean;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < 16; ++w) mean += sh[w];
            *a.loss = (float)(mean / a.P);
        }
    }
}

// Gradient of the logits from the row statistics: coef[row / rows_per_coef] (* *alpha) ([v == y] - exp(x - m) / s).
// A row whose factor is zero is not read.
template <typename T>
__global__ __launch_bounds__(256) void logprob_bwd_kernel(const T* logits, long ld, const int64_t* __restrict__ labels, const float* __restrict__ stats,
                                                          const float* __restrict__ coef, int rows_per_coef, const float* __restrict__ alpha, T* dlogits,
                                                          long ldd, int W, int V, int R) {
    constexpr int NT = 256, U = 4;
    if (block_index() >= R) return;
    const int tid = threadIdx.x, row = R - 1 - (int)block_index();
    const int64_t y = labels[row];
    T* const d = dlogits + (long)row * ldd;
    const T* x = logits + (long)row * ld;
    const bool counted = y >= 0 && y < V;
    float c0 = 0.f;
    if (counted) {
        c0 = coef[row / rows_per_coef];
        if (alpha != nullptr) c0 *= *alpha;
    }
    if (c0 == 0.f) {
        const float z[kPer<T>] = {};
        for (long c = (long)tid * kPer<T>; c < W; c += NT * kPer<T>) store_chunk(d, (int)c, W, z);
        return;
    }
    const float m = stats[2 * (long)row], cs = -c0 / stats[2 * (long)row + 1];
    for (long c0i = (long)tid * kPer<T>; c0i < V; c0i += (long)U * NT * kPer<T>) {
        u32x4_t reg[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long c = c0i + (long)u * NT * kPer<T>;
            if (c < V) reg[u] = load_chunk<T, true>(x, (int)c, V);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long c = c0i + (long)u * NT * kPer<T>;
            if (c < V) {
                float f[kPer<T>];
                unpack<T>(reg[u], f);
#pragma unroll
                for (int k = 0; k < kPer<T>; ++k) f[k] = cs * grad_exp<T>(f[k] - m);
                if (y >= c && y < c + kPer<T>) {
#pragma unroll
                    for (int k = 0; k < kPer<T>; ++k)
                        if (c + k == y) f[k] += c0;
                }
                store_chunk(d, (int)c, V, f);
            }
        }
    }
    zero_cols<T, NT>(d, V, W);
}

// out[j] = sum of x[j * n .. (j + 1) * n) / per, in 64 bits (terms of either sign may leave little)
__global__ __launch_bounds__(1024) void rows_mean_kernel(const float* __restrict__ x, long n, long per, float* __restrict__ out) {
    __shared__ double sh[16];
    double s = 0.0;
    for (long i = threadIdx.x; i < n; i += 1024) s += x[(long)blockIdx.x * n + i];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) s += sh[w];
        out[blockIdx.x] = (float)(s / per);
    }
}

// counts[i]: counted tokens of sequence i (seq) or of the i-th of kCountParts equal stretches of the batch
__global__ __launch_bounds__(256) void count_kernel(const int64_t* __restrict__ labels, long R, long per, int V, int* __restrict__ counts, long slots) {
    __shared__ int sh[4];
    if (block_index() >= slots) return;
    const long lo = block_index() * per, hi = lo + per < R ? lo + per : R;
    int n = 0;
    for (long i = lo + threadIdx.x; i < hi; i += 256) { const int64_t y = labels[i]; n += y >= 0 && y < V; }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) counts[block_index()] = sh[0] + sh[1] + sh[2] + sh[3];
}

// The policy loss from log-probabilities that are there already (the two-step form): coef per row and the terms
__global__ __launch_bounds__(256) void policy_terms_kernel(const float* __restrict__ logp, const int64_t* __restrict__ labels, int V, PolicyArgs p, float* __restrict__ coef) {
    const long R = (long)p.N * p.T, row = (long)blockIdx.x * 256 + threadIdx.x;
    float w = 0.f;
    if (!p.seq_mean) w = policy_weight(p, 0, threadIdx.x & 63);       // the wave sums the stretches together
    if (row >= R) return;
    const int64_t y = labels[row];
    float t[3] = {0.f, 0.f, 0.f}, c = 0.f;
    if (y >= 0 && y < V) {
        if (p.seq_mean) w = policy_weight(p, (int)row, 0);
        c = policy_token(p, (int)row, logp[row], w, t);
    }
    coef[row] = c;
    p.terms[row] = t[0];
    p.terms[R + row] = t[1];
    p.terms[2 * R + row] = t[2];
}

// Threads and chunks of a row: the smallest workgroup whose registers hold it, so that short rows keep many rows in flight on a CU
// and a BART row (50,265 bf16 logits: 512 threads x 13 chunks, 52 registers; f32: 1024 x 13) is resident as a whole.  Scoring | policy loss, us, against
// the next larger workgroup: 8,192 x 2,000 8 | 21 (35 | 53), 4,096 x 16,000 24 | 54 (55 | 175), 4,096 x 50,265 88 | 177 (207 | 289).
template <typename T, bool POLICY>
int launch_rows(const RowArgs<T>& a, hipStream_t s) {
    const dim3 g = grid_of(a.R);
    const long chunks = ((long)a.V + kPer<T> - 1) / kPer<T>;
    if (chunks <= 64 * 4) hipLaunchKernelGGL((row_kernel<T, 64, 4, POLICY>), g, dim3(64), 0, s, a);
    else if (chunks <= 256 * 8) hipLaunchKernelGGL((row_kernel<T, 256, 8, POLICY>), g, dim3(256), 0, s, a);
    else if (chunks <= 512 * 13) hipLaunchKernelGGL((row_kernel<T, 512, 13, POLICY>), g, dim3(512), 0, s, a);
    else if (chunks <= 1024 * 13) hipLaunchKernelGGL((row_kernel<T, 1024, 13, POLICY>), g, dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((long_row_kernel<T, POLICY>), g, dim3(1024), 0, s, a);
    return ok();
}

bool bad_rows(long R, int V, long ld) { return R <= 0 || R > 0x7fffffffL || V <= 0 || V > 0x7fffffff - 16384 || ld < V; }
bool bad_align(int dtype, const void* p) { return ((uintptr_t)p & (dtype == MMSUM_BF16 ? 1 : 3)) != 0; }

template <typename T>
RowArgs<T> row_args(const void* logits, long ld, const int64_t* labels, int R, int V, float* logp, float* stats) {
    RowArgs<T> a = {};
    a.logits = static_cast<const T*>(logits); a.ld = ld; a.labels = labels; a.R = R; a.V = V; a.logp = logp; a.stats = stats;
    return a;
}

template <typename T>
int launch_bwd(const void* logits, long ld, const int64_t* labels, const float* stats, const float* coef, int rows_per_coef, const float* alpha, void* dlogits,
               long ldd, int W, int V, int R, hipStream_t s) {
    hipLaunchKernelGGL((logprob_bwd_kernel<T>), grid_of(R), dim3(256), 0, s, static_cast<const T*>(logits), ld, labels, stats, coef, rows_per_coef, alpha,
                       static_cast<T*>(dlogits), ldd, W, V, R);
    return ok();
}

long count_slots(int N, int seq_mean) { return seq_mean ? N : kCountParts; }
int launch_counts(const int64_t* labels, int N, int T, int V, int seq_mean, int* counts, hipStream_t s) {
    const long R = (long)N * T, per = seq_mean ? T : (R + kCountParts - 1) / kCountParts;
    hipLaunchKernelGGL(count_kernel, grid_of(count_slots(N, seq_mean)), dim3(256), 0, s, labels, R, per, V, counts, count_slots(N, seq_mean));
    return ok();
}

}  // namespace

extern "C" int mmsum_token_logprob(int dtype, const void* logits, long ld, const int64_t* labels, float* logp, float* stats, int R, int V, void* stream) {
    if (bad_rows(R, V, ld)) return MMSUM_ERR_BAD_SHAPE;
    if (dtype != MMSUM_BF16 && dtype != MMSUM_F32) return MMSUM_ERR_BAD_DTYPE;
    if (any_null(logits, labels, logp) || bad_align(dtype, logits)) return MMSUM_ERR_BAD_ALIGN;
    if (dtype == MMSUM_BF16) return launch_rows<bf16_t, false>(row_args<bf16_t>(logits, ld, labels, R, V, logp, stats), (hipStream_t)stream);
    return launch_rows<float, false>(row_args<float>(logits, ld, labels, R, V, logp, stats), (hipStream_t)stream);
}

extern "C" int mmsum_token_logprob_bwd(int dtype, const void* logits, long ld, const int64_t* labels, const float* stats, const float* coef, int rows_per_coef,
                                       const float* alpha, void* dlogits, long ldd, int W, int R, int V, void* stream) {
    if (bad_rows(R, V, ld) || rows_per_coef <= 0 || W < V || W > 0x7fffffff - 16384 || ldd < W) return MMSUM_ERR_BAD_SHAPE;
    if (dtype != MMSUM_BF16 && dtype != MMSUM_F32) return MMSUM_ERR_BAD_DTYPE;
    if (any_null(logits, labels, stats, coef, dlogits) || bad_align(dtype, logits) || bad_align(dtype, dlogits)) return MMSUM_ERR_BAD_ALIGN;
    if (dtype == MMSUM_BF16) return launch_bwd<bf16_t>(logits, ld, labels, stats, coef, rows_per_coef, alpha, dlogits, ldd, W, V, R, (hipStream_t)stream);
    return launch_bwd<float>(logits, ld, labels, stats, coef, rows_per_coef, alpha, dlogits, ldd, W, V, R, (hipStream_t)stream);
}

extern "C" int mmsum_sequence_logprob(const float* logp, const int64_t* labels, int N, int T, int V, int average, float* out, void* stream) {
    if (N <= 0 || T <= 0 || V <= 0 || (long)N * T > 0x7fffffffL) return MMSUM_ERR_BAD_SHAPE;
    if (any_null(logp, labels, out)) return MMSUM_ERR_BAD_ALIGN;
    hipLaunchKernelGGL(sequence_sum_kernel, grid_of((N + 3L) / 4), dim3(256), 0, (hipStream_t)stream, logp, labels, N, T, V, average, out);
    return ok();
}

extern "C" int mmsum_preference_pairs(const float* logp, const int64_t* labels, const float* ref, int P, int T, int V, float beta, float smoothing, int average,
                                      float* seq, float* margins, float* pair_loss, float* coef, float* loss, void* stream) {
    if (P <= 0 || T <= 0 || V <= 0 || 2L * P * T > 0x7fffffffL || !(smoothing >= 0.f && smoothing <= 1.f)) return MMSUM_ERR_BAD_SHAPE;
    if (any_null(logp, labels, seq, margins, pair_loss, coef, loss)) return MMSUM_ERR_BAD_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    PairArgs a = {logp, labels, ref, P, T, V, average, beta, smoothing, seq, margins, pair_loss, coef, loss};
    // one workgroup, a wave a pair, with the mean (us, this | two launches: 1 x 33 3.2 | 4.7, 16 x 128 4.5 | 5.4; in turns 36 x 32 6.4 | 5.2, 128 x 256 28 | 6.5)
    if (P <= 16) {
        hipLaunchKernelGGL(pair_kernel, dim3(1), dim3(1024), 0, s, a);
    } else {
        a.loss = nullptr;
        hipLaunchKernelGGL(pair_kernel, grid_of((P + 3L) / 4), dim3(256), 0, s, a);
        hipLaunchKernelGGL(rows_mean_kernel, dim3(1), dim3(1024), 0, s, pair_loss, (long)P, (long)P, loss);
    }
    return ok();
}

// workspace: logp [2PT], stats [2PT][2], pair_loss [P], coef [2P]
extern "C" long mmsum_preference_workspace(int P, int T) { return P <= 0 || T <= 0 ? 0 : (6L * P * T + 3L * P) * (long)sizeof(float); }
extern "C" int mmsum_preference_loss(int dtype, const void* logits, long ld, const int64_t* labels, const float* ref, int P, int T, int V, float beta, float smoothing,
                                     int average, float* loss, float* margins, float* seq, void* dlogits, long ldd, int W, void* workspace, void* stream) {
    if (P <= 0 || T <= 0 || bad_rows(2L * P * T, V, ld) || W < V || W > 0x7fffffff - 16384 || ldd < W || !(smoothing >= 0.f && smoothing <= 1.f)) return MMSUM_ERR_BAD_SHAPE;
    if (dtype != MMSUM_BF16 && dtype != MMSUM_F32) return MMSUM_ERR_BAD_DTYPE;
    if (workspace == nullptr) return MMSUM_ERR_WORKSPACE;
    if (any_null(logits, labels, loss, margins, seq, dlogits) || bad_align(dtype, logits) || bad_align(dtype, dlogits) || ((uintptr_t)workspace & 15)) return MMSUM_ERR_BAD_ALIGN;
    const int R = 2 * P * T;
    float* const logp = static_cast<float*>(workspace);
    float* const stats = logp + R;
    float* const pair_loss = stats + 2L * R;
    float* const coef = pair_loss + P;
    hipStream_t s = (hipStream_t)stream;
    // Statistics, the pairs, then the gradient from the last row to the first.  All rows but the last 400 MB are read past the caches, which leaves those
    // to the second reading.  The memory-side cache holds 256 MB, and rows that do not count are not read: 400 MB are 256 where 64 % count, between a full
    // batch, for which less were better, and a ragged one, for which more were.  Measured (us; every row past the caches | all but the last 256 MB | 400 | 512 |
    // none past; bf16, 128 x 50,265 a sequence), 36 pairs: all counted 497 | 477 | 481 | 484 | 488, 84 % 456 | 429 | 427 | 427 | 435, 51 % 362 | 338 | 324 | 317 |
    // 316; 18 pairs: 261 | 240 | 241 | 242 | 242, 84 % 240 | 215 | 211 | 211 | 211, 51 % 193 | 168 | 155 | 152 | 152; 72 pairs: 975 | 953 | 965 | 969 | 992, 84 % 879 |
    // 855 | 854 | 855 | 876, 51 % 693 | 669 | 656 | 650 | 653; f32, 18 pairs: 588 | 565 | 566 | 567 | 569, 84 % 543 | 515 | 510 | 510 | 514, 51 % 423 | 407 | 387 |
    // 377 | 373; the gradient's memory reused or fresh alike.  (Every row's workgroup of the gradient taking its pair's sums itself in place of the pairs'
    // launch: 4 x 128 x 1,009 equal, 36 x 128 x 1,009 30 -> 52 us.)
    const auto run = [&](auto of_type) {
        typedef decltype(of_type) T_;
        RowArgs<T_> a = row_args<T_>(logits, ld, labels, R, V, logp, stats);
        const long keep = (400L << 20) / (ld * (long)sizeof(T_));
        a.past = keep < R ? R - (int)keep : 0;
        int rc = launch_rows<T_, false>(a, s);
        if (rc == MMSUM_OK) rc = mmsum_preference_pairs(logp, labels, ref, P, T, V, beta, smoothing, average, seq, margins, pair_loss, coef, loss, stream);
        return rc == MMSUM_OK ? launch_bwd<T_>(logits, ld, labels, stats, coef, T, nullptr, dlogits, ldd, W, V, R, s) : rc;
    };
    return dtype == MMSUM_BF16 ? run(bf16_t{}) : run(float{});
}

// workspace: terms [3][NT], counts
extern "C" long mmsum_policy_workspace(int N, int T) {
    return N <= 0 || T <= 0 ? 0 : 3L * N * T * (long)sizeof(float) + (long)(N > kCountParts ? N : kCountParts) * (long)sizeof(int);
}
// Rows of the logits count their sequence (or the small batch) themselves, under the latency of the row: a launch less (us, V = 1,009, this | a launch:
// token mean 3 x 57 7.2 | 9.1, 8 x 128 9.7 | 9.9, 16 x 128 13.1 | 11.4; sequence mean 4 x 128 7.4 | 8.8, 4 x 1,024 14.1 | 14.0, 4 x 4,096 56 | 31)
static bool rows_count(int N, int T, int seq_mean) { return seq_mean ? T <= 1024 : (long)N * T <= 1024; }
static int policy_setup(PolicyArgs& p, const int64_t* labels, int V, const float* old_logp, const float* ref_logp, const float* adv, int adv_per_token, int N, int T, float clip_low,
                        float clip_high, float kl_coef, int seq_mean, void* workspace) {
    if (!(clip_low >= 0.f) || !(clip_high >= 0.f) || kl_coef != kl_coef) return MMSUM_ERR_BAD_SHAPE;
    if (workspace == nullptr) return MMSUM_ERR_WORKSPACE;
    if (any_null(labels, old_logp, adv) || ((uintptr_t)workspace & 15)) return MMSUM_ERR_BAD_ALIGN;
    p.labels = labels; p.V = V;
    p.old_logp = old_logp; p.ref_logp = ref_logp; p.adv = adv;
    p.terms = static_cast<float*>(workspace);
    p.counts = reinterpret_cast<int*>(p.terms + 3L * N * T);
    p.adv_per_token = adv_per_token; p.seq_mean = seq_mean; p.N = N; p.T = T;
    p.lo = 1.f - clip_low; p.hi = 1.f + clip_high; p.kl_coef = kl_coef;
    return MMSUM_OK;
}

extern "C" int mmsum_policy_terms(const float* logp, const int64_t* labels, const float* old_logp, const float* ref_logp, const float* adv, int adv_per_token, int N,
                                  int T, int V, float clip_low, float clip_high, float kl_coef, int seq_mean, float* out, float* coef, void* workspace, void* stream) {
    if (N <= 0 || T <= 0 || V <= 0 || (long)N * T > 0x7fffffffL) return MMSUM_ERR_BAD_SHAPE;
    if (any_null(logp, out, coef)) return MMSUM_ERR_BAD_ALIGN;
    PolicyArgs p = {};
    int rc = policy_setup(p, labels, V, old_logp, ref_logp, adv, adv_per_token, N, T, clip_low, clip_high, kl_coef, seq_mean, workspace);
    hipStream_t s = (hipStream_t)stream;
    const long R = (long)N * T;
    if (rc == MMSUM_OK) rc = launch_counts(labels, N, T, V, seq_mean, const_cast<int*>(p.counts), s);
    if (rc != MMSUM_OK) return rc;
    hipLaunchKernelGGL(policy_terms_kernel, dim3((unsigned)((R + 255) / 256)), dim3(256), 0, s, logp, labels, V, p, coef);
    hipLaunchKernelGGL(rows_mean_kernel, dim3(3), dim3(1024), 0, s, p.terms, R, 1L, out);
    return ok();
}

extern "C" int mmsum_policy_loss(int dtype, const void* logits, long ld, const int64_t* labels, const float* old_logp, const float* ref_logp, const float* adv,
                                 int adv_per_token, int N, int T, int V, float clip_low, float clip_high, float kl_coef, int seq_mean, float* out, float* logp,
                                 void* dlogits, long ldd, int W, void* workspace, void* stream) {
    if (N <= 0 || T <= 0 || bad_rows((long)N * T, V, ld) || W < V || W > 0x7fffffff - 16384 || ldd < W) return MMSUM_ERR_BAD_SHAPE;
    if (dtype != MMSUM_BF16 && dtype != MMSUM_F32) return MMSUM_ERR_BAD_DTYPE;
    if (any_null(logits, out, logp, dlogits) || bad_align(dtype, logits) || bad_align(dtype, dlogits)) return MMSUM_ERR_BAD_ALIGN;
    PolicyArgs p = {};
    int rc = policy_setup(p, labels, V, old_logp, ref_logp, adv, adv_per_token, N, T, clip_low, clip_high, kl_coef, seq_mean, workspace);
    hipStream_t s = (hipStream_t)stream;
    const int R = N * T;
    if (rows_count(N, T, seq_mean)) p.counts = nullptr;
    else if (rc == MMSUM_OK) rc = launch_counts(labels, N, T, V, seq_mean, const_cast<int*>(p.counts), s);
    if (rc != MMSUM_OK) return rc;
    if (dtype == MMSUM_BF16) {
        RowArgs<bf16_t> a = row_args<bf16_t>(logits, ld, labels, R, V, logp, nullptr);
        a.dlogits = static_cast<bf16_t*>(dlogits); a.ldd = ldd; a.W = W; a.pol = p;
        rc = launch_rows<bf16_t, true>(a, s);
    } else {
        RowArgs<float> a = row_args<float>(logits, ld, labels, R, V, logp, nullptr);
        a.dlogits = static_cast<float*>(dlogits); a.ldd = ldd; a.W = W; a.pol = p;
        rc = launch_rows<float, true>(a, s);
    }
    if (rc != MMSUM_OK) return rc;
    hipLaunchKernelGGL(rows_mean_kernel, dim3(3), dim3(1024), 0, s, p.terms, (long)R, 1L, out);
    return ok();
}
