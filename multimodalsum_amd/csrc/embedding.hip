// Embedding lookup with scaling, y[i] = scale E[ids[i]], and the table's gradient dE[v] = scale sum of dy[i] over ids[i] == v.
//
// The gradient goes by SORTED tokens: a stable radix sort brings equal ids together in batch order (few ids: every workgroup lists those of its
// own rows), fixed stretches of the sorted list are summed each by one wave, and a token's stretches are added in order -- no floating-point
// atomics, so a gradient is the same bit for bit on every run, and a frequent token (padding excluded, still a few percent of a text) is
// summed by many waves at once.
// Ids outside 0 .. V-1 read as zero rows and leave no gradient, and so does pad_id in the gradient.
// Bound: HBM (dy once, dE once).
#include "entry_checks.h"
#include "mmsum_device.h"
#include "mmsum_kernels.h"

namespace {

inline int ok() { return hipGetLastError() == hipSuccess ? MMSUM_OK : MMSUM_ERR_HIP; }

// ---- lookup ------------------------------------------------------------------------------------------------------------------------
// VEC elements a thread and step; tpr threads a row (a power of two <= 256), 256 / tpr rows at a time, ROWS of them in flight
template <typename T, int VEC> struct Vec;
template <> struct Vec<bf16_t, 8> { typedef u32x4_t type; };
template <> struct Vec<float, 4> { typedef u32x4_t type; };
typedef int i32x4_t __attribute__((ext_vector_type(4)));
template <> struct Vec<bf16_t, 1> { typedef bf16_t type; };
template <> struct Vec<float, 1> { typedef float type; };

constexpr int kFwdRows = 8;
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const int64_t* __restrict__ ids, const T* __restrict__ E, long lde, T* __restrict__ y, long ldy, long n,
                                                        int V, int D, float scale, int tpr_log2) {
    constexpr int ROWS = kFwdRows;
    const int tpr = 1 << tpr_log2, rpb = 256 >> tpr_log2;
    const int c0 = ((int)threadIdx.x & (tpr - 1)) * VEC;
    const long r0 = block_index() * (rpb * ROWS) + (threadIdx.x >> tpr_log2);
    int64_t id[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) id[j] = r0 + j * rpb < n ? ids[r0 + j * rpb] : -1;
    for (int c = c0; c < D; c += tpr * VEC) {
        typename Vec<T, VEC>::type v[ROWS];
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
            if (id[j] >= 0 && id[j] < V) v[j] = *reinterpret_cast<const typename Vec<T, VEC>::type*>(E + (long)id[j] * lde + c);
            else v[j] = typename Vec<T, VEC>::type{};
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
            if (r0 + j * rpb < n) {
                T t[VEC];
                __builtin_memcpy(t, &v[j], sizeof(t));
#pragma unroll
                for (int k = 0; k < VEC; ++k) t[k] = from_f32<T>(to_f32(t[k]) * scale);
                __builtin_memcpy(&v[j], t, sizeof(t));
                __builtin_nontemporal_store(v[j], reinterpret_cast<typename Vec<T, VEC>::type*>(y + (r0 + j * rpb) * ldy + c));
            }
    }
}

// ---- sort --------------------------------------------------------------------------------------------------------------------------
// Least-significant-digit radix sort of (key, position), 8 bits a pass.  A key is the id, or V for a position without a gradient (sorted
// behind every id).  A pass is stable: within a tile a wave's rounds keep their order, tiles keep theirs.
__device__ __forceinline__ uint32_t key_of(int64_t id, int V, int64_t pad_id) { return id >= 0 && id < V && id != pad_id ? (uint32_t)id : (uint32_t)V; }

// lanes of the wave whose digit equals this lane's (among the `act` lanes)
__device__ __forceinline__ uint64_t same_digit(uint32_t d, uint64_t act) {
    uint64_t m = act;
#pragma unroll
    for (int b = 0; b < 8; ++b) {
        const uint64_t v = __ballot((d >> b) & 1);
        m &= (d >> b) & 1 ? v : ~v;
    }
    return m;
}

// One round: every active lane of the wave gets its rank among the equal digits this wave has met (cnt: the wave's 256 counters)
__device__ __forceinline__ int wave_rank(volatile int* cnt, uint32_t d, bool active, int lane) {
    const uint64_t act = __ballot(active);
    const uint64_t same = same_digit(d, act);
    int base = 0;
    if (active) base = cnt[d];
    __builtin_amdgcn_wave_barrier();
    const int before = __popcll(same & ((1ull << lane) - 1));
    if (active && before == 0) cnt[d] = base + __popcll(same);
    __builtin_amdgcn_wave_barrier();
    return base + before;
}

constexpr int kSub = 1024;               // elements a workgroup ranks at a time (four rounds of its four waves)
constexpr int kMaxTiles = 256;
constexpr long kHistBytes = (long)kMaxTiles * 256 * 4;

// hist[tile][256]: digits of every tile.  (Counting a later pass's digits with atomics while the pass in front of it places the elements
// saves a launch and was slower: the frequent ids meet in a few counters, 14 -> 28 us at 147,456 ids.)
template <bool FIRST>
__global__ __launch_bounds__(256) void sort_hist_kernel(const int64_t* __restrict__ ids, const uint32_t* __restrict__ keys, int n, int tile, int V, int64_t pad_id, int shift,
                                                        int* __restrict__ hist) {
    __shared__ int h[256];
    h[threadIdx.x] = 0;
    __syncthreads();
    const long lo = (long)blockIdx.x * tile, hi = lo + tile < n ? lo + tile : n;
    for (long i = lo + threadIdx.x; i < hi; i += 256) atomicAdd(&h[((FIRST ? key_of(ids[i], V, pad_id) : keys[i]) >> shift) & 255], 1);
    __syncthreads();
    hist[blockIdx.x * 256 + threadIdx.x] = h[threadIdx.x];
}

// moves a tile's elements to their places: in front of a digit's elements of this tile come all smaller digits and the earlier tiles' equal ones
template <bool FIRST>
__global__ __launch_bounds__(256) void sort_scatter_kernel(const int64_t* __restrict__ ids, const uint32_t* __restrict__ keys, const int* __restrict__ pos, int n, int tile,
                                                           int tiles, int V, int64_t pad_id, int shift, const int* __restrict__ hist, uint32_t* __restrict__ okeys,
                                                           int* __restrict__ opos) {
    __shared__ __attribute__((aligned(16))) int cnt[4][256], wbase[4][256];
    __shared__ int wsum[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long lo = (long)blockIdx.x * tile, hi = lo + tile < n ? lo + tile : n;
    uint32_t key[4];
    int from[4];
    auto load = [&](long base) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const long i = base + wave * 256 + r * 64 + lane;
            key[r] = i < hi ? (FIRST ? key_of(ids[i], V, pad_id) : keys[i]) : 0u;
            from[r] = FIRST ? (int)i : i < hi ? pos[i] : 0;
        }
    };
    load(lo);                                                      // under way beside the counts
    // the digits' totals and what earlier tiles hold of them: a wave sums every fourth tile, four digits a lane, 16 requests at a time (all
    // tiles after one another by the digit's own thread were most of the kernel)
    {
        i32x4_t sum = {0, 0, 0, 0}, front = {0, 0, 0, 0};
        for (int t0 = wave; t0 < tiles; t0 += 64) {
            i32x4_t v[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) v[u] = t0 + 4 * u < tiles ? *reinterpret_cast<const i32x4_t*>(hist + (t0 + 4 * u) * 256 + 4 * lane) : i32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                if (t0 + 4 * u < (int)blockIdx.x) front += v[u];
                sum += v[u];
            }
        }
        *reinterpret_cast<i32x4_t*>(&cnt[wave][4 * lane]) = sum;
        *reinterpret_cast<i32x4_t*>(&wbase[wave][4 * lane]) = front;
    }
    __syncthreads();
    const int total = cnt[0][tid] + cnt[1][tid] + cnt[2][tid] + cnt[3][tid], before = wbase[0][tid] + wbase[1][tid] + wbase[2][tid] + wbase[3][tid];
    int incl = total;                                              // inclusive scan over the digits
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 3; ++w)
        if (w < wave) incl += wsum[w];
    int off = incl - total + before;                              // this digit's next place
    for (long base = lo; base < hi; base += kSub) {
#pragma unroll
        for (int w = 0; w < 4; ++w) cnt[w][tid] = 0;
        __syncthreads();
        int rank[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) rank[r] = wave_rank(cnt[wave], (key[r] >> shift) & 255, base + wave * 256 + r * 64 + lane < hi, lane);
        __syncthreads();
        {
            int o = off;
#pragma unroll
            for (int w = 0; w < 4; ++w) { wbase[w][tid] = o; o += cnt[w][tid]; }
            off = o;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (base + wave * 256 + r * 64 + lane < hi) {
                const int p = wbase[wave][(key[r] >> shift) & 255] + rank[r];
                okeys[p] = key[r];
                opos[p] = from[r];
            }
        if (base + kSub < hi) load(base + kSub);
        __syncthreads();
    }
}

// The whole sort of up to 4096 ids in one workgroup's LDS: one launch for two passes' four (gradient of 4,096 ids into 50,265 x 1,024 50 us, by the
// passes 56; into 70,000 x 64 31 | 38).
constexpr int kSmall = 4096;
__global__ __launch_bounds__(1024) void sort_small_kernel(const int64_t* __restrict__ ids, int n, int V, int64_t pad_id, int bits, uint32_t* __restrict__ okeys, int* __restrict__ opos) {
    __shared__ uint32_t lk[2][kSmall];
    __shared__ uint16_t lp[2][kSmall];
    __shared__ int cnt[16][256];
    __shared__ int scan[256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < n; i += 1024) { lk[0][i] = key_of(ids[i], V, pad_id); lp[0][i] = (uint16_t)i; }
    int cur = 0;
    for (int shift = 0; shift < bits; shift += 8) {
        for (int i = tid; i < 16 * 256; i += 1024) (&cnt[0][0])[i] = 0;
        __syncthreads();
        uint32_t key[4];
        int rank[4], p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = wave * 256 + r * 64 + lane;
            const bool act = i < n;
            key[r] = act ? lk[cur][i] : 0u;
            p[r] = act ? lp[cur][i] : 0;
            rank[r] = wave_rank(cnt[wave], (key[r] >> shift) & 255, act, lane);
        }
        __syncthreads();
        int total = 0;
        if (tid < 256) {
            for (int w = 0; w < 16; ++w) { const int v = cnt[w][tid]; cnt[w][tid] = total; total += v; }
            scan[tid] = total;
        }
        __syncthreads();
        for (int o = 1; o < 256; o <<= 1) {
            const int v = tid < 256 && tid >= o ? scan[tid - o] : 0;
            __syncthreads();
            if (tid < 256) scan[tid] += v;
            __syncthreads();
        }
        if (tid < 256) scan[tid] -= total;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (wave * 256 + r * 64 + lane < n) {
                const int d = (key[r] >> shift) & 255, o = scan[d] + cnt[wave][d] + rank[r];
                lk[cur ^ 1][o] = key[r];
                lp[cur ^ 1][o] = (uint16_t)p[r];
            }
        cur ^= 1;
        __syncthreads();
    }
    for (int i = tid; i < n; i += 1024) { okeys[i] = lk[cur][i]; opos[i] = lp[cur][i]; }
}

// ---- up to 2048 ids: one launch ----------------------------------------------------------------------------------------------------
// A workgroup takes up to four neighbouring rows of the table (8 KB of them) and clears them at once, which needs no id and keeps the memory
// busy while they arrive.  It reads every id, lists the positions that name a row of its own in batch order, and writes those rows' sums over
// the zeros.  A row is summed by tpr threads of four columns (VEC = 1: one), its positions in order, eight requested at a time.  Reading all ids
// in every workgroup is cheap while they are few (1,152 ids: 9 KB from L2); the launches and waits of a sort are not.  More rows a workgroup
// put a text's most frequent tokens, neighbours in the table, into one.  Measured (MI355X, bf16, table 50,265 x 1,024, its clearing alone 31 us):
// 1,152 ids 37 us (16 KB a workgroup 38, 4 KB 48); 2,048 ids 38 us (42, 58).  From there on by sorting (3,000 ids 59 us): with lists of 4,096 fewer
// workgroups fit a CU, 57 us at 1,152 ids and 66 at 3,000.
constexpr int kFew = 2048, kRowsMax = 4;
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_bwd_few_kernel(const T* __restrict__ dy, long lddy, const int64_t* __restrict__ ids, int n, int V, int D, float scale, int64_t pad_id,
                                                            int accumulate, float* __restrict__ dE, int rows, int tpr_log2) {
    constexpr int R = kFew / 256;                                      // rounds of the workgroup over the ids
    __shared__ uint16_t list[kRowsMax][kFew];                          // positions of a row
    __shared__ int at[kRowsMax][R * 4], count[kRowsMax];               // of a round and wave: entries of a row, then those in front of them
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long v0 = block_index() * rows;
    if (v0 >= V) return;
    const int here = (int)(V - v0 < rows ? V - v0 : rows);
    int64_t all[R];
#pragma unroll
    for (int i = 0; i < R; ++i) all[i] = i * 256 + tid < n ? ids[i * 256 + tid] : -1;
    if (!accumulate) {
        float* const z = dE + v0 * D;
        const long cells = (long)here * D, quads = ((uintptr_t)z & 15) == 0 ? cells / 4 : 0;
        for (long i = tid; i < quads; i += 256) __builtin_nontemporal_store(f32x4_t{0.f, 0.f, 0.f, 0.f}, reinterpret_cast<f32x4_t*>(z) + i);
        for (long i = quads * 4 + tid; i < cells; i += 256) z[i] = 0.f;
    }
    int row[R];                                                        // this thread's ids: the row in the workgroup's range, or -1
    bool any = false;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        row[i] = all[i] >= v0 && all[i] < v0 + here && all[i] != pad_id ? (int)(all[i] - v0) : -1;
        any |= row[i] >= 0;
    }
    if (!__syncthreads_or(any)) return;                                // none of the rows is named: most stretches of a large table
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                   // the zeros are in front of the sums (other waves' too: barriers follow)
    int before[R];                                                     // lanes of the wave in front with the same row
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int r = 0; r < kRowsMax; ++r) {
            const uint64_t m = __ballot(row[i] == r);
            if (row[i] == r) before[i] = __popcll(m & ((1ull << lane) - 1));
            if (lane == 0) at[r][i * 4 + wave] = __popcll(m);
        }
    __syncthreads();
    static_assert(kRowsMax * R * 4 <= 256 && R * 4 == 32, "a half wave scans a row's counts");
    if (tid < kRowsMax * R * 4) {
        const int r = tid >> 5, j = tid & 31, c = at[r][j];
        int sum = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up(sum, o, 32);
            sum += j >= o ? v : 0;
        }
        at[r][j] = sum - c;
        if (j == 31) count[r] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (row[i] >= 0) list[row[i]][at[row[i]][i * 4 + wave] + before[i]] = (uint16_t)(i * 256 + tid);
    __syncthreads();
    constexpr int AHEAD = 8;
    const int tpr = 1 << tpr_log2, groups = 256 >> tpr_log2;
    for (int r = tid >> tpr_log2; r < here; r += groups) {
        const int hi = count[r];
        if (hi == 0) continue;
        for (int c = (tid & (tpr - 1)) * VEC; c < D; c += tpr * VEC) {
            float acc[VEC] = {};
            for (int i0 = 0; i0 < hi; i0 += AHEAD) {
                float f[AHEAD][VEC];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const T* const src = dy + (long)list[r][i0 + u < hi ? i0 + u : 0] * lddy + c;
                    if constexpr (VEC == 1) f[u][0] = to_f32(*src);
                    else if constexpr (sizeof(T) == 2) {
                        const bf16x4_t t = *reinterpret_cast<const bf16x4_t*>(src);
#pragma unroll
                        for (int k = 0; k < 4; ++k) f[u][k] = (float)t[k];
                    } else {
                        const f32x4_t t = *reinterpret_cast<const f32x4_t*>(src);
#pragma unroll
                        for (int k = 0; k < 4; ++k) f[u][k] = t[k];
                    }
                }
#pragma unroll
                for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) acc[k] += i0 + u < hi ? f[u][k] : 0.f;
            }
            float* const o = dE + (v0 + r) * D + c;
            if constexpr (VEC == 1) *o = accumulate ? *o + scale * acc[0] : scale * acc[0];
            else {
                f32x4_t s = {scale * acc[0], scale * acc[1], scale * acc[2], scale * acc[3]};
                if (accumulate) s += *reinterpret_cast<f32x4_t*>(o);
                *reinterpret_cast<f32x4_t*>(o) = s;
            }
        }
    }
}
template <typename T>
int embed_bwd_few(const void* dy, long lddy, const int64_t* ids, int n, int V, int D, float scale, int64_t pad_id, int accumulate, float* dE, hipStream_t s) {
    const bool vec = D % 4 == 0 && lddy % 4 == 0 && ((uintptr_t)dy & (4 * sizeof(T) - 1)) == 0 && ((uintptr_t)dE & 15) == 0;
    const int rows = D <= 2048 / kRowsMax ? kRowsMax : D <= 1024 ? 2 : 1, steps = vec ? D / 4 : D;
    int lg = 0;
    while ((1 << lg) < steps && lg < 8) ++lg;
    const dim3 grid = grid_of((V + (long)rows - 1) / rows);
    if (vec) hipLaunchKernelGGL((embed_bwd_few_kernel<T, 4>), grid, dim3(256), 0, s, (const T*)dy, lddy, ids, n, V, D, scale, pad_id, accumulate, dE, rows, lg);
    else hipLaunchKernelGGL((embed_bwd_few_kernel<T, 1>), grid, dim3(256), 0, s, (const T*)dy, lddy, ids, n, V, D, scale, pad_id, accumulate, dE, rows, lg);
    return ok();
}

// ---- sums --------------------------------------------------------------------------------------------------------------------------
// A wave sums a stretch of 8, 16 or 32 sorted positions over 512 columns (eight a lane).  A token whose positions all lie in the stretch is
// finished; a token that crosses its ends leaves partial sums: part[stretch][0] of the one that began before it, part[stretch][1] of the
// one that begins in it and goes on (stretch_join_kernel adds those up).
constexpr int kCols = 512;
// Positions of a stretch: few of them while that is what keeps the card busy, more where the partial sums' traffic and the joins' length count.
// Whole gradient, bf16, a text's token frequencies into 50,265 x 1,024, us in stretches of 8 | 16 | 32: 3,000 ids 58 | - | 76, 9,216 69 | 73 | 83,
// 20,000 81 | 77 | 86, 40,000 107 | 99 | 93, 147,456 293 | 200 | 172
int stretch_of(long n) { return n <= 16384 ? 8 : n <= 32768 ? 16 : 32; }

// eight columns of a lane: VEC: neighbours, else 64 apart
template <typename T, bool VEC> __device__ __forceinline__ void load8(const T* __restrict__ row, int c, int D, int lane, float (&f)[8]) {
    if constexpr (VEC) {
        if (c < D) {
            if constexpr (sizeof(T) == 2) {
                T t[8];
                const u32x4_t v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(row + c));
                __builtin_memcpy(t, &v, 16);
#pragma unroll
                for (int k = 0; k < 8; ++k) f[k] = to_f32(t[k]);
            } else {
                const f32x4_t a = __builtin_nontemporal_load(reinterpret_cast<const f32x4_t*>(row + c)), b = __builtin_nontemporal_load(reinterpret_cast<const f32x4_t*>(row + c + 4));
#pragma unroll
                for (int k = 0; k < 4; ++k) { f[k] = a[k]; f[4 + k] = b[k]; }
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (c + k * 64 < D) f[k] = to_f32(row[c + k * 64]);
    }
}
template <bool VEC> __device__ __forceinline__ void store8(float* __restrict__ row, int c, int D, const float (&f)[8], float scale, bool accumulate) {
    if constexpr (VEC) {
        if (c < D) {
            f32x4_t* const o = reinterpret_cast<f32x4_t*>(row + c);
            f32x4_t a = {scale * f[0], scale * f[1], scale * f[2], scale * f[3]}, b = {scale * f[4], scale * f[5], scale * f[6], scale * f[7]};
            if (accumulate) { a += o[0]; b += o[1]; }
            o[0] = a;
            o[1] = b;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int cc = c + k * 64;
            if (cc < D) row[cc] = accumulate ? row[cc] + scale * f[k] : scale * f[k];
        }
    }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void stretch_sum_kernel(const T* __restrict__ dy, long lddy, const uint32_t* __restrict__ keys, const int* __restrict__ pos, int n, int sl, int V, int D,
                                                          float scale, int accumulate, float* __restrict__ part, float* __restrict__ dE) {
    const int lane = threadIdx.x & 63;
    // the column blocks of a stretch on neighbouring waves: the rows' halves are asked for together
    const int cols = (D + kCols - 1) / kCols;
    const long idx = block_index() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long st = idx / cols, lo = st * sl;
    if (lo >= n) return;
    const int len = (int)(n - lo < sl ? n - lo : sl);
    const int col0 = (int)(idx - st * cols) * kCols, c = VEC ? col0 + lane * 8 : col0 + lane;
    const int Dc = VEC ? D : (D < col0 + kCols ? D : col0 + kCols);
    // the stretch's keys and positions ride on the lanes; lanes 62 / 63 hold the neighbours in front and behind
    uint32_t k = (uint32_t)V;
    int p = 0;
    if (lane < len) { k = keys[lo + lane]; p = pos[lo + lane]; }
    if (lane == 62 && lo > 0) k = keys[lo - 1];
    if (lane == 63 && lo + len < n) k = keys[lo + len];
    if ((uint32_t)__builtin_amdgcn_readlane(k, 0) >= (uint32_t)V) return;      // behind every id
    if (k >= (uint32_t)V) p = __builtin_amdgcn_readlane(p, 0);                // requested with the others, never added
    const uint32_t kbefore = lo > 0 ? (uint32_t)__builtin_amdgcn_readlane(k, 62) : 0xffffffffu;
    const uint32_t kbehind = lo + len < n ? (uint32_t)__builtin_amdgcn_readlane(k, 63) : 0xffffffffu;
    float acc[8] = {};
    constexpr int AHEAD = 8;
    float f[AHEAD][8] = {};
    bool open = false;                                             // the current token began before the stretch
    for (int i0 = 0; i0 < len; i0 += AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            load8<T, VEC>(dy + (long)__builtin_amdgcn_readlane(p, i0 + u) * lddy, c, Dc, lane, f[u]);
        }
        // all of them back before the first store: a wait between the stores below would be for the stores (one row at a time, 25 us of it at 1,152 ids)
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(f[u][e]));
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int i = i0 + u;
            if (i >= len) break;
            const uint32_t key = __builtin_amdgcn_readlane(k, i);
            if (key >= (uint32_t)V) return;                        // sorted behind every id: nothing more to sum
            const uint32_t prev = i > 0 ? (uint32_t)__builtin_amdgcn_readlane(k, i - 1) : kbefore;
            const uint32_t next = i + 1 < len ? (uint32_t)__builtin_amdgcn_readlane(k, i + 1) : kbehind;
            if (i == 0) open = key == prev;
            else if (key != prev) open = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = key != prev || i == 0 ? f[u][e] : acc[e] + f[u][e];
            if (key != next || i + 1 == len) {
                const bool goes_on = key == next;
                if (!open && !goes_on) store8<VEC>(dE + (long)key * D, c, Dc, acc, scale, accumulate != 0);
                else store8<VEC>(part + (st * 2 + (open ? 0 : 1)) * D, c, Dc, acc, 1.f, false);
            }
        }
    }
}

// Rows of the table that no id names: zeros.  A wave takes 16 neighbouring rows, its lanes bisect the sorted keys for them.
__device__ __forceinline__ void clear_absent(const uint32_t* __restrict__ keys, int n, int V, int D, float* __restrict__ dE, long v0) {
    const int lane = threadIdx.x & 63;
    if (v0 >= V) return;
    const uint32_t v = (uint32_t)(v0 + (lane & 15));
    int a = 0, b = n;
    while (a < b) {
        const int mid = (int)(((long)a + b) / 2);
        if (keys[mid] < v) a = mid + 1;
        else b = mid;
    }
    const uint64_t absent = __ballot(!(a < n && keys[a] == v));
    for (int r = 0; r < 16 && v0 + r < V; ++r) {
        if (!((absent >> r) & 1)) continue;
        float* const row = dE + (v0 + r) * D;
        if (D % 4 == 0 && ((uintptr_t)dE & 15) == 0) {
            for (int c = lane * 4; c < D; c += 256) *reinterpret_cast<f32x4_t*>(row + c) = f32x4_t{0.f, 0.f, 0.f, 0.f};
        } else {
            for (int c = lane; c < D; c += 64) row[c] = 0.f;
        }
    }
}

// A token that begins in stretch st and goes on: part[st][1] + part[st + 1][0] + ... in order.  One workgroup a stretch, a thread four
// columns (VEC: as one vector), up to AHEAD stretches requested at a time: the most frequent tokens of a text (a few per cent of it, over a
// hundred stretches) are the kernel's tail.  Workgroups from `joins` on clear the absent rows: the joins wait for memory, the clearing fills it.
template <bool VEC>
__global__ __launch_bounds__(256) void stretch_join_kernel(const uint32_t* __restrict__ keys, int n, int sl, int V, int D, float scale, int accumulate, const float* __restrict__ part,
                                                           float* __restrict__ dE, int joins) {
    if (block_index() >= joins) {
        if (!accumulate) clear_absent(keys, n, V, D, dE, ((block_index() - joins) * 4 + (threadIdx.x >> 6)) * 16);
        return;
    }
    constexpr int AHEAD = 16;
    const int lane = threadIdx.x & 63;
    const long st = block_index(), begin = st * sl, end = begin + sl;      // end < n: the grid leaves the last stretch out
    // five keys at once: the last of the stretch and the first behind it, the first and the one in front, the next stretch's last
    const uint32_t key = keys[end - 1], behind = keys[end], first = keys[begin], front = keys[begin > 0 ? begin - 1 : 0];
    long b = end + sl < n ? end + sl : n;
    const uint32_t far = keys[b - 1];
    if (key >= (uint32_t)V || behind != key || (begin > 0 && first == key && front == key)) return;      // nothing goes on, or it began earlier
    long last = st + 1;
    if (far == key && b < n) {                                     // beyond the next stretch, perhaps: the token's last stretch in [lo, lo + len), 64 probes a step
        long lo = st + 1, len = (n + sl - 1) / sl - lo;
        while (len > 1) {
            const long step = (len + 63) / 64, q = lo + (lane + 1) * step;           // does the token reach stretch q?
            const uint64_t reach = __ballot(q < lo + len && keys[q * sl < n ? q * sl : n - 1] == key);
            const int r = __popcll(reach);                                           // sorted: the lanes that say yes come first
            const long nlo = lo + r * step;
            len = lo + len - nlo < step ? lo + len - nlo : step;
            lo = nlo;
        }
        last = lo;
    }
    for (int c = (int)threadIdx.x * 4; c < D; c += 1024) {
        f32x4_t s = {0.f, 0.f, 0.f, 0.f};
        for (long q0 = st; q0 <= last; q0 += AHEAD) {
            f32x4_t f[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                f[u] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                if (q0 + u <= last) {
                    const float* const row = part + ((q0 + u) * 2 + (q0 + u == st ? 1 : 0)) * D;
                    if constexpr (VEC) f[u] = *reinterpret_cast<const f32x4_t*>(row + c);
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (c + e < D) f[u][e] = row[c + e];
                }
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) s += f[u];
        }
        float* const o = dE + (long)key * D + c;
        if constexpr (VEC) {
            f32x4_t r = s * scale;
            if (accumulate) r += *reinterpret_cast<f32x4_t*>(o);
            *reinterpret_cast<f32x4_t*>(o) = r;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < D) o[e] = accumulate ? o[e] + scale * s[e] : scale * s[e];
        }
    }
}

template <typename T>
int embed_fwd_t(const int64_t* ids, const void* E, long lde, void* y, long ldy, long n, int V, int D, float scale, hipStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    const bool vec = D % VEC == 0 && lde % VEC == 0 && ldy % VEC == 0 && (((uintptr_t)E | (uintptr_t)y) & 15) == 0;
    const int steps = vec ? D / VEC : D;
    int lg = 0;
    while ((1 << lg) < steps && lg < 8) ++lg;
    const long blocks = (n + kFwdRows * (256 >> lg) - 1) / (kFwdRows * (256 >> lg));
    if (blocks > 1L << 36) return MMSUM_ERR_BAD_SHAPE;               // (the second axis holds 2^15 rows of workgroups)
    if (vec) hipLaunchKernelGGL((embed_fwd_kernel<T, VEC>), grid_of(blocks), dim3(256), 0, s, ids, (const T*)E, lde, (T*)y, ldy, n, V, D, scale, lg);
    else hipLaunchKernelGGL((embed_fwd_kernel<T, 1>), grid_of(blocks), dim3(256), 0, s, ids, (const T*)E, lde, (T*)y, ldy, n, V, D, scale, lg);
    return ok();
}

struct SortPlan { int tile, tiles; };
SortPlan sort_plan(int n) {
    const int subs = (int)(((long)n + kSub - 1) / kSub), per = (subs + kMaxTiles - 1) / kMaxTiles;
    return SortPlan{per * kSub, (subs + per - 1) / per};
}
long align16(long b) { return (b + 15) & ~15L; }

template <typename T>
int embed_bwd_t(const void* dy, long lddy, const int64_t* ids, int n, int V, int D, float scale, int64_t pad_id, int accumulate, float* dE, char* ws, hipStream_t s) {
    if (n <= kFew) return embed_bwd_few<T>(dy, lddy, ids, n, V, D, scale, pad_id, accumulate, dE, s);
    const long nb = align16((long)n * 4);
    uint32_t* k0 = reinterpret_cast<uint32_t*>(ws);
    int* p0 = reinterpret_cast<int*>(ws + nb);
    uint32_t* k1 = reinterpret_cast<uint32_t*>(ws + 2 * nb);
    int* p1 = reinterpret_cast<int*>(ws + 3 * nb);
    int* hist = reinterpret_cast<int*>(ws + 4 * nb);
    float* part = reinterpret_cast<float*>(ws + 4 * nb + kHistBytes);
    int bits = 0;
    while (bits < 32 && ((uint32_t)V >> bits) != 0) ++bits;
    if (n <= kSmall) {
        hipLaunchKernelGGL(sort_small_kernel, dim3(1), dim3(1024), 0, s, ids, n, V, pad_id, bits, k0, p0);
    } else {
        const SortPlan sp = sort_plan(n);
        const dim3 g(sp.tiles);
        for (int shift = 0; shift < bits; shift += 8) {
            if (shift == 0) {
                hipLaunchKernelGGL((sort_hist_kernel<true>), g, dim3(256), 0, s, ids, nullptr, n, sp.tile, V, pad_id, shift, hist);
                hipLaunchKernelGGL((sort_scatter_kernel<true>), g, dim3(256), 0, s, ids, nullptr, nullptr, n, sp.tile, sp.tiles, V, pad_id, shift, hist, k0, p0);
            } else {
                hipLaunchKernelGGL((sort_hist_kernel<false>), g, dim3(256), 0, s, ids, k0, n, sp.tile, V, pad_id, shift, hist);
                hipLaunchKernelGGL((sort_scatter_kernel<false>), g, dim3(256), 0, s, ids, k0, p0, n, sp.tile, sp.tiles, V, pad_id, shift, hist, k1, p1);
                uint32_t* tk = k0; k0 = k1; k1 = tk;
                int* tp = p0; p0 = p1; p1 = tp;
            }
        }
    }
    const int sl = stretch_of(n);
    const long stretches = ((long)n + sl - 1) / sl;
    const long waves = stretches * ((D + kCols - 1) / kCols);
    const bool vec = D % 8 == 0 && lddy % (16 / (int)sizeof(T)) == 0 && (((uintptr_t)dy | (uintptr_t)dE) & 15) == 0;
    const dim3 grid = grid_of((waves + 3) / 4);
    if (vec) hipLaunchKernelGGL((stretch_sum_kernel<T, true>), grid, dim3(256), 0, s, (const T*)dy, lddy, k0, p0, n, sl, V, D, scale, accumulate, part, dE);
    else hipLaunchKernelGGL((stretch_sum_kernel<T, false>), grid, dim3(256), 0, s, (const T*)dy, lddy, k0, p0, n, sl, V, D, scale, accumulate, part, dE);
    const long joins = ((long)n - 1) / sl;                    // stretches with another one behind them
    const long jn = joins + (accumulate ? 0 : (V + 63L) / 64);
    if (jn == 0) return ok();
    const dim3 jg = grid_of(jn);
    if (vec) hipLaunchKernelGGL((stretch_join_kernel<true>), jg, dim3(256), 0, s, k0, n, sl, V, D, scale, accumulate, part, dE, (int)joins);
    else hipLaunchKernelGGL((stretch_join_kernel<false>), jg, dim3(256), 0, s, k0, n, sl, V, D, scale, accumulate, part, dE, (int)joins);
    return ok();
}

__global__ __launch_bounds__(256) void zero_kernel(float* __restrict__ p, long n) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) p[i] = 0.f;
}

}  // namespace

extern "C" int mmsum_embed_fwd(int dtype, const int64_t* ids, const void* E, long lde, void* y, long ldy, long n, int V, int D, float scale, void* stream) {
    if (n <= 0 || V <= 0 || D <= 0 || lde < D || ldy < D) return MMSUM_ERR_BAD_SHAPE;
    if (any_null(ids, E, y)) return MMSUM_ERR_BAD_ALIGN;
    if (dtype == MMSUM_BF16) return ((uintptr_t)E | (uintptr_t)y) & 1 ? MMSUM_ERR_BAD_ALIGN : embed_fwd_t<bf16_t>(ids, E, lde, y, ldy, n, V, D, scale, (hipStream_t)stream);
    if (dtype == MMSUM_F32) return ((uintptr_t)E | (uintptr_t)y) & 3 ? MMSUM_ERR_BAD_ALIGN : embed_fwd_t<float>(ids, E, lde, y, ldy, n, V, D, scale, (hipStream_t)stream);
    return MMSUM_ERR_BAD_DTYPE;
}

extern "C" long mmsum_embed_bwd_workspace(long n, int D) {
    if (n <= kFew || n > 0x3fffffffL || D <= 0) return 0;              // few ids need none
    return 4 * align16(n * 4) + kHistBytes + (n + stretch_of(n) - 1) / stretch_of(n) * 2 * D * (long)sizeof(float);
}
extern "C" int mmsum_embed_bwd(int dtype, const void* dy, long lddy, const int64_t* ids, long n, int V, int D, float scale, int64_t pad_id, int accumulate, float* dE,
                               void* workspace, void* stream) {
    if (n < 0 || n > 0x3fffffffL || V <= 0 || V > 0x7ffffff0 || D <= 0 || lddy < D) return MMSUM_ERR_BAD_SHAPE;
    if (dtype != MMSUM_BF16 && dtype != MMSUM_F32) return MMSUM_ERR_BAD_DTYPE;
    if (n > kFew && workspace == nullptr) return MMSUM_ERR_WORKSPACE;
    if (dE == nullptr || (n > 0 && any_null(dy, ids)) || ((uintptr_t)workspace & 15) || ((uintptr_t)dE & 3) || ((uintptr_t)dy & (dtype == MMSUM_BF16 ? 1 : 3))) return MMSUM_ERR_BAD_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    if (n == 0) {
        if (!accumulate) hipLaunchKernelGGL(zero_kernel, dim3(1024), dim3(256), 0, s, dE, (long)V * D);
        return ok();
    }
    if (dtype == MMSUM_BF16) return embed_bwd_t<bf16_t>(dy, lddy, ids, (int)n, V, D, scale, pad_id, accumulate, dE, static_cast<char*>(workspace), s);
    return embed_bwd_t<float>(dy, lddy, ids, (int)n, V, D, scale, pad_id, accumulate, dE, static_cast<char*>(workspace), s);
}
