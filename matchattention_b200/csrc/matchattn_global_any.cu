// Dense attention on the ordinary arithmetic units: float32, and head widths and alignments that the matrix kernels do not take.
//
// A block of 16 x 16 threads owns a tile of query rows of one key head (the g query heads that share it side by side: row
// r is query r / g of head r % g, so K and V are read once for all of them) and walks the keys.  Tiles lie in shared memory
// channel by channel ([channel][row], rows 16 bytes aligned, pitch + 4), so that a thread of the score product reads its rows and
// its keys as 16-byte words per channel and the value product reads four keys of a channel at once.  All sums are float32.
// Bound by the multiply-add rate and the shared-memory reads behind it (a thread of a 128-row block reads three 16-byte words per
// 32 multiply-adds of a score).  Measured, one B200, float32: 2 x 1000 tokens, 8 heads x 128 266 us (31 TFLOP/s); the training
// step 1340, of which dK and dV 660 and dQ 405: slower than a library's products over a stored score matrix (858) at that size.
// Single tokens, 3 items of 8000 keys, 16 heads x 128 on 4 key heads 110 us (0.9 TB/s; a warp's loads of 16 bytes lie in 32 rows).
//
// A value that no row of a tile may see can still be infinite or NaN, and 0 * NaN is NaN: a tile that holds such a value is
// accumulated term by term, leaving out the hidden terms.
#include "matchattn_global_mma.cuh"

#include <type_traits>

namespace matchattn {
namespace {

constexpr int kAnyThreads = 256;

template <typename T>
__device__ __forceinline__ void load_four(const T *p, int n, bool vec, float (&x)[4])
{
    if (vec && n >= 4) {
        if constexpr (sizeof(T) == 4) {
            const float4 t = *reinterpret_cast<const float4 *>(p);
            x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
        } else {
            const uint2 t = *reinterpret_cast<const uint2 *>(p);
            x[0] = DT<T>::unpack(t.x, 0), x[1] = DT<T>::unpack(t.x, 1), x[2] = DT<T>::unpack(t.y, 0), x[3] = DT<T>::unpack(t.y, 1);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = i < n ? load_one<T>(p + i) : 0.0f;
    }
}

// A tile of ROWS rows between global and shared memory, in registers: four channels of a row at a time.  Fetched ahead of its place
// in shared memory falling free, it is on its way while the tile before it is computed.
template <typename T, int DP, int ROWS>
struct Tile {
    static constexpr int kPieces = (ROWS * (DP / 4) + kAnyThreads - 1) / kAnyThreads;
    float x[kPieces][4];

    // rows that `row` has no address for, and channels from d on, are zero
    template <typename Row>
    __device__ __forceinline__ void fetch(int d, bool vec, Row row)
    {
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const int i = threadIdx.x + k * kAnyThreads, r = i % ROWS, c = i / ROWS * 4;
            const T *src = i < ROWS * (DP / 4) && c < d ? row(r) : nullptr;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[k][j] = 0.0f;
            if (src != nullptr) load_four<T>(src + c, d - c, vec, x[k]);
        }
    }

    // dst[channel][row]; true if a value is infinite or NaN
    __device__ __forceinline__ bool put(float *dst) const
    {
        bool bad = false;
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const int i = threadIdx.x + k * kAnyThreads, r = i % ROWS, c = i / ROWS * 4;
            if (i >= ROWS * (DP / 4)) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                bad |= !(fabsf(x[k][j]) <= 3.402823466e38f);
                dst[(c + j) * (ROWS + 4) + r] = x[k][j];
            }
        }
        return bad;
    }
};

template <typename T, int DP, int ROWS, typename Row>
__device__ __forceinline__ bool load_transposed(float *dst, int d, bool vec, Row row)
{
    Tile<T, DP, ROWS> tile;
    tile.fetch(d, vec, row);
    return tile.put(dst);
}

template <int R>
__device__ __forceinline__ void read_run(const float *p, float (&x)[R])
{
    if constexpr (R == 8) {
        const float4 t = *reinterpret_cast<const float4 *>(p), u = *reinterpret_cast<const float4 *>(p + 4);
        x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w, x[4] = u.x, x[5] = u.y, x[6] = u.z, x[7] = u.w;
    } else if constexpr (R == 4) {
        const float4 t = *reinterpret_cast<const float4 *>(p);
        x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
    } else if constexpr (R == 2) {
        const float2 t = *reinterpret_cast<const float2 *>(p);
        x[0] = t.x, x[1] = t.y;
    } else {
        x[0] = *p;
    }
}

// s[i][j] += sum over the channels of a[channel][RA * ty + i] * b[channel][RB * tx + j]
template <int RA, int RB, int PA, int PB>
__device__ __forceinline__ void products(float (&s)[RA][RB], const float *a, const float *b, int d, int ty, int tx)
{
    a += RA * ty;
    b += RB * tx;
#pragma unroll 4
    for (int c = 0; c < d; ++c) {
        float x[RA], y[RB];
        read_run<RA>(a + c * PA, x);
        read_run<RB>(b + c * PB, y);
#pragma unroll
        for (int i = 0; i < RA; ++i)
#pragma unroll
            for (int j = 0; j < RB; ++j) s[i][j] = fmaf(x[i], y[j], s[i][j]);
    }
}

// acc[i][c] += sum over the K columns of w[RA * ty + i][column] * b[tx + 16 c][column]; with `bad` only over those that seen(i, column)
template <int RA, int NC, int K, typename Seen>
__device__ __forceinline__ void accumulate(float (&acc)[RA][NC], const float *w, const float *b, int ty, int tx, bool bad, Seen seen)
{
    constexpr int P = K + 4;
    w += RA * ty * P;
    b += tx * P;
    if (!bad) {
#pragma unroll 2
        for (int j = 0; j < K; j += 4) {
            float4 x[RA];
#pragma unroll
            for (int i = 0; i < RA; ++i) x[i] = *reinterpret_cast<const float4 *>(w + i * P + j);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float4 y = *reinterpret_cast<const float4 *>(b + 16 * c * P + j);
#pragma unroll
                for (int i = 0; i < RA; ++i)
                    acc[i][c] = fmaf(x[i].w, y.w, fmaf(x[i].z, y.z, fmaf(x[i].y, y.y, fmaf(x[i].x, y.x, acc[i][c]))));
            }
        }
        return;
    }
    for (int j = 0; j < K; ++j) {
#pragma unroll
        for (int i = 0; i < RA; ++i) {
            const float x = w[i * P + j];
            if (!seen(i, j)) continue;
#pragma unroll
            for (int c = 0; c < NC; ++c) acc[i][c] = fmaf(x, b[16 * c * P + j], acc[i][c]);
        }
    }
}

// tanh(x / cap) of every element in place, for products x / scale.  (A block takes the polynomial where all of a warp's scores are well
// below the cap; the library's function is long, and a copy of it per element.)
template <int RA, int RB>
__device__ __forceinline__ void capped(float (&s)[RA][RB], float inverse_cap)
{
    float big = 0.0f;
#pragma unroll
    for (int i = 0; i < RA; ++i)
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            s[i][j] *= inverse_cap;
            big = fmaxf(big, fabsf(s[i][j]));
        }
    if (__all_sync(0xffffffffu, big <= kSmallTanh)) {
#pragma unroll
        for (int i = 0; i < RA; ++i)
#pragma unroll
            for (int j = 0; j < RB; ++j) s[i][j] = tanh_small(s[i][j]);
    } else {
#pragma unroll
        for (int i = 0; i < RA; ++i)
#pragma unroll
            for (int j = 0; j < RB; ++j) s[i][j] = tanh_one(s[i][j]);
    }
}

struct RowOf {
    int n, head;
};

// Row r of key head kh, of the g heads from h_begin on that are walked.
__device__ __forceinline__ RowOf row_of(const GlobalParams &p, int kh, int r, int g, int h_begin)
{
    const int n = r / g;
    return {n, kh * p.g + h_begin + r - n * g};
}

__device__ __forceinline__ RowOf row_of(const GlobalParams &p, int kh, int r) { return row_of(p, kh, r, p.g, 0); }

template <typename T>
__device__ __forceinline__ const T *at(const void *base, const long long (&s)[3], int b, int n, int head)
{
    return static_cast<const T *>(base) + b * s[0] + n * s[1] + head * s[2];
}

// lowest and highest document of the block's rows, in shared memory
__device__ __forceinline__ void row_documents(const GlobalParams &p, int b, int r0, int rows, int *range)
{
    if (threadIdx.x == 0) range[0] = 0x7fffffff, range[1] = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < rows; i += kAnyThreads) {
        const int n = (r0 + i) / p.g;
        if (n >= p.N) continue;
        const int doc = p.q_docs[static_cast<long long>(b) * p.N + n];
        if (doc < 0) continue;
        atomicMin(range, doc);
        atomicMax(range + 1, doc);
    }
    __syncthreads();
}

template <typename T, int DP, int RM, int RN>
__global__ void __launch_bounds__(kAnyThreads) global_any_forward_kernel(const GlobalParams p)
{
    chain_begin();
    constexpr int BM = 16 * RM, BN = 16 * RN, PM = BM + 4, PN = BN + 4, NC = DP / 16;
    extern __shared__ __align__(16) float smem[];
    float *qt = smem, *kvt = qt + DP * PM, *w = kvt + DP * PN;
    float2 *place = reinterpret_cast<float2 *>(w + BM * PN);
    int *doc = reinterpret_cast<int *>(place + BN), *range = doc + BN;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    // (the last queries of a causal call see most: they begin first)
    const int r0 = (gridDim.x - 1 - blockIdx.x) * BM, kh = blockIdx.y, b = blockIdx.z % p.B, split = blockIdx.z / p.B;
    const int rows = p.N * p.g;
    const GlobalMask mask = global_mask(p, b);

    load_transposed<T, DP, BM>(qt, p.d, p.vec, [&](int r) -> const T * {
        if (r0 + r >= rows) return nullptr;
        const RowOf t = row_of(p, kh, r0 + r);
        return at<T>(p.q, p.qs, b, t.n, t.head);
    });
    if (p.q_docs) row_documents(p, b, r0, BM, range);

    float acc[RM][NC] = {}, top[RM], sum[RM], slope[RM];
    float2 here[RM];
    int n_of[RM], doc_of[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int r = min(r0 + RM * ty + i, rows - 1);
        const RowOf t = row_of(p, kh, r);
        top[i] = -INFINITY;
        sum[i] = 0.0f;
        n_of[i] = t.n;
        slope[i] = p.slopes ? p.slopes[t.head] * kLog2e : 0.0f;
        here[i] = map_place(t.n + mask.shift, p.width);
        doc_of[i] = p.q_docs ? p.q_docs[static_cast<long long>(b) * p.N + t.n] : 0;
    }
    const int end = key_end(mask, (min(r0 + BM, rows) - 1) / p.g);
    const int whole = p.q_docs ? -1 : key_end(mask, r0 / p.g);         // tiles that end below it are seen by all rows
    const int t_end = p.splits > 1 ? min((end + BN - 1) / BN, (split + 1) * p.tiles_per_split) : (end + BN - 1) / BN;
    Tile<T, DP, BN> tile;
    const auto fetch = [&](const void *base, const long long (&stride)[3], int j0) {
        tile.fetch(p.d, p.vec, [&](int r) -> const T * { return j0 + r < mask.len ? at<T>(base, stride, b, j0 + r, kh) : nullptr; });
    };
    const int t_begin = split * p.tiles_per_split;
    if (!p.k_docs && t_begin < t_end) fetch(p.k, p.ks, t_begin * BN);
    for (int t = t_begin; t < t_end; ++t) {
        const int j0 = t * BN;
        __syncthreads();
        bool any = true;
        if (tid < BN) {
            const int j = j0 + tid;
            place[tid] = map_place(j, p.width);
            if (p.k_docs) {
                const int dk = j < p.M ? p.k_docs[static_cast<long long>(b) * p.M + j] : -1;
                doc[tid] = dk;
                any = dk >= range[0] && dk <= range[1];
            }
        } else if (p.k_docs) {
            any = false;
        }
        if (p.k_docs) {
            if (!__syncthreads_or(any)) continue;
            fetch(p.k, p.ks, j0);
        }
        tile.put(kvt);
        __syncthreads();
        fetch(p.v, p.vs, j0);
        float s[RM][RN] = {};
        products<RM, RN, PM, PN>(s, qt, kvt, p.d, ty, tx);
        // scores in units of log2; what only some calls or tiles have stands in loops of its own
        if (p.cap != 0.0f) capped(s, p.scale / p.cap);
        const float unit = (p.cap != 0.0f ? p.cap : p.scale) * kLog2e;
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < RN; ++j) s[i][j] *= unit;
        if (p.slopes) {
#pragma unroll
            for (int j = 0; j < RN; ++j) {
                const float2 there = place[RN * tx + j];
#pragma unroll
                for (int i = 0; i < RM; ++i) s[i][j] -= slope[i] * map_distance(here[i], there);
            }
        }
        if (j0 + BN > whole) {
#pragma unroll
            for (int j = 0; j < RN; ++j) {
                const int c = RN * tx + j, id = p.k_docs ? doc[c] : 0;
#pragma unroll
                for (int i = 0; i < RM; ++i)
                    if (!sees(mask, n_of[i], j0 + c) || id != doc_of[i] || id < 0) s[i][j] = -INFINITY;
            }
        }
        float high[RM];
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            high[i] = top[i];
#pragma unroll
            for (int j = 0; j < RN; ++j) high[i] = fmaxf(high[i], s[i][j]);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) high[i] = fmaxf(high[i], __shfl_xor_sync(0xffffffffu, high[i], o));
            const float ref = high[i] == -INFINITY ? 0.0f : high[i];
            const float shrink = exp2_fast(top[i] - ref);
            top[i] = high[i];
            sum[i] *= shrink;
#pragma unroll
            for (int c = 0; c < NC; ++c) acc[i][c] *= shrink;
#pragma unroll
            for (int j = 0; j < RN; ++j) {
                const float e = exp2_fast(s[i][j] - ref);
                sum[i] += e;
                w[(RM * ty + i) * PN + RN * tx + j] = e;
            }
        }
        __syncthreads();
        const bool bad = __syncthreads_or(tile.put(kvt));
        if (!p.k_docs && t + 1 < t_end) fetch(p.k, p.ks, j0 + BN);
        accumulate<RM, NC, BN>(acc, w, kvt, ty, tx, bad, [&](int i, int c) {
            const int id = p.k_docs ? doc[c] : 0;
            return sees(mask, n_of[i], j0 + c) && id == doc_of[i] && id >= 0;
        });
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
        const int r = r0 + RM * ty + i;
        if (r >= rows) continue;
        const RowOf t = row_of(p, kh, r);
        const float inv = sum[i] == 0.0f ? 0.0f : 1.0f / sum[i];
        const bool empty = sum[i] == 0.0f;
        const long long row = (static_cast<long long>(b) * p.h + t.head) * p.N + t.n;
        const float lse = top[i] + log2f(sum[i]);
        if (p.splits > 1) {
            const long long part = static_cast<long long>(split) * p.B * p.h * p.N + row;
            if (tx == 0) p.part_lse[part] = empty ? -INFINITY : lse;
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (tx + 16 * c < p.d) p.part_out[part * p.d + tx + 16 * c] = empty ? 0.0f : acc[i][c] * inv;
        } else {
            if (p.lse && tx == 0) p.lse[row] = empty ? INFINITY : lse;
            const long long out = ((static_cast<long long>(b) * p.N + t.n) * p.h + t.head) * p.d;
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (tx + 16 * c < p.d) store_result<T>(p, out + tx + 16 * c, empty ? 0.0f : acc[i][c] * inv);
        }
    }
}

// dQ: the rows of the forward kernel, scores and probabilities recomputed.  K and V take turns in one place, K twice.
template <typename T, int DP, int RM, int RN>
__global__ void __launch_bounds__(kAnyThreads) global_any_dq_kernel(const GlobalParams p)
{
    chain_begin();
    constexpr int BM = 16 * RM, BN = 16 * RN, PM = BM + 4, PN = BN + 4, NC = DP / 16;
    extern __shared__ __align__(16) float smem[];
    float *qt = smem, *dot = qt + DP * PM, *kvt = dot + DP * PM, *w = kvt + DP * PN;
    float2 *place = reinterpret_cast<float2 *>(w + BM * PN);
    int *doc = reinterpret_cast<int *>(place + BN), *range = doc + BN;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    // (the last queries of a causal call see most: they begin first)
    const int r0 = (gridDim.x - 1 - blockIdx.x) * BM, kh = blockIdx.y, b = blockIdx.z, rows = p.N * p.g;
    const GlobalMask mask = global_mask(p, b);
    load_transposed<T, DP, BM>(qt, p.d, p.vec, [&](int r) -> const T * {
        if (r0 + r >= rows) return nullptr;
        const RowOf t = row_of(p, kh, r0 + r);
        return at<T>(p.q, p.qs, b, t.n, t.head);
    });
    load_transposed<T, DP, BM>(dot, p.d, p.vec, [&](int r) -> const T * {
        if (r0 + r >= rows) return nullptr;
        const RowOf t = row_of(p, kh, r0 + r);
        return static_cast<const T *>(p.d_out) + ((static_cast<long long>(b) * p.N + t.n) * p.h + t.head) * p.d;
    });
    if (p.q_docs) row_documents(p, b, r0, BM, range);
    float acc[RM][NC] = {}, lse[RM], delta[RM], slope[RM];
    float2 here[RM];
    int n_of[RM], doc_of[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const RowOf t = row_of(p, kh, min(r0 + RM * ty + i, rows - 1));
        const long long row = (static_cast<long long>(b) * p.h + t.head) * p.N + t.n;
        lse[i] = p.lse[row];
        delta[i] = p.delta[row];
        n_of[i] = t.n;
        slope[i] = p.slopes ? p.slopes[t.head] * kLog2e : 0.0f;
        here[i] = map_place(t.n + mask.shift, p.width);
        doc_of[i] = p.q_docs ? p.q_docs[static_cast<long long>(b) * p.N + t.n] : 0;
    }
    const int end = key_end(mask, (min(r0 + BM, rows) - 1) / p.g);
    const int whole = p.q_docs ? -1 : key_end(mask, r0 / p.g);         // tiles that end below it are seen by all rows
    Tile<T, DP, BN> tile;
    const auto fetch = [&](const void *base, const long long (&stride)[3], int j0) {
        tile.fetch(p.d, p.vec, [&](int r) -> const T * { return j0 + r < mask.len ? at<T>(base, stride, b, j0 + r, kh) : nullptr; });
    };
    if (!p.k_docs && end > 0) fetch(p.k, p.ks, 0);
    for (int j0 = 0; j0 < end; j0 += BN) {
        __syncthreads();
        bool any = true;
        if (tid < BN) {
            const int j = j0 + tid;
            place[tid] = map_place(j, p.width);
            if (p.k_docs) {
                const int dk = j < p.M ? p.k_docs[static_cast<long long>(b) * p.M + j] : -1;
                doc[tid] = dk;
                any = dk >= range[0] && dk <= range[1];
            }
        } else if (p.k_docs) {
            any = false;
        }
        if (p.k_docs) {
            if (!__syncthreads_or(any)) continue;
            fetch(p.k, p.ks, j0);
        }
        tile.put(kvt);
        __syncthreads();
        fetch(p.v, p.vs, j0);
        float s[RM][RN] = {}, dp[RM][RN] = {};
        products<RM, RN, PM, PN>(s, qt, kvt, p.d, ty, tx);
        __syncthreads();
        tile.put(kvt);
        __syncthreads();
        fetch(p.k, p.ks, j0);
        products<RM, RN, PM, PN>(dp, dot, kvt, p.d, ty, tx);
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < RN; ++j) dp[i][j] -= delta[i];
        if (p.cap != 0.0f) {
            capped(s, p.scale / p.cap);
#pragma unroll
            for (int i = 0; i < RM; ++i)
#pragma unroll
                for (int j = 0; j < RN; ++j) dp[i][j] *= fmaf(-s[i][j], s[i][j], 1.0f);
        }
        const float unit = (p.cap != 0.0f ? p.cap : p.scale) * kLog2e;
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < RN; ++j) s[i][j] *= unit;
        if (p.slopes) {
#pragma unroll
            for (int j = 0; j < RN; ++j) {
                const float2 there = place[RN * tx + j];
#pragma unroll
                for (int i = 0; i < RM; ++i) s[i][j] -= slope[i] * map_distance(here[i], there);
            }
        }
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < RN; ++j) dp[i][j] *= exp2_fast(s[i][j] - lse[i]);
        if (j0 + BN > whole) {
#pragma unroll
            for (int j = 0; j < RN; ++j) {
                const int c = RN * tx + j, id = p.k_docs ? doc[c] : 0;
#pragma unroll
                for (int i = 0; i < RM; ++i)
                    if (!sees(mask, n_of[i], j0 + c) || id != doc_of[i] || id < 0) dp[i][j] = 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < RN; ++j) w[(RM * ty + i) * PN + RN * tx + j] = dp[i][j];
        __syncthreads();
        const bool bad = __syncthreads_or(tile.put(kvt));
        if (!p.k_docs && j0 + BN < end) fetch(p.k, p.ks, j0 + BN);
        accumulate<RM, NC, BN>(acc, w, kvt, ty, tx, bad, [&](int i, int c) {
            const int id = p.k_docs ? doc[c] : 0;
            return sees(mask, n_of[i], j0 + c) && id == doc_of[i] && id >= 0;
        });
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int r = r0 + RM * ty + i;
        if (r >= rows) continue;
        const RowOf t = row_of(p, kh, r);
        T *out = static_cast<T *>(p.d_q) + ((static_cast<long long>(b) * p.N + t.n) * p.h + t.head) * p.d;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (tx + 16 * c < p.d) store_one<T>(out + tx + 16 * c, acc[i][c] * p.scale);
    }
}

// dK and dV: a block owns a tile of keys of one key head and walks the query rows of all heads that share it.  Q and dO take turns
// in one place, Q twice.
template <typename T, int DP, int RM, int RN>
__global__ void __launch_bounds__(kAnyThreads) global_any_dkv_kernel(const GlobalParams p)
{
    chain_begin();
    constexpr int BM = 16 * RM, BN = 16 * RN, PM = BM + 4, PN = BN + 4, NC = DP / 16;
    extern __shared__ __align__(16) float smem[];
    float *kt = smem, *vt = kt + DP * PM, *qot = vt + DP * PM, *w = qot + DP * PN;
    float2 *place = reinterpret_cast<float2 *>(w + BM * PN);
    float *lse = reinterpret_cast<float *>(place + BN), *delta = lse + BN, *slope = delta + BN;
    int *n_of = reinterpret_cast<int *>(slope + BN), *doc = n_of + BN, *range = doc + BN;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int j0 = blockIdx.x * BM, kh = blockIdx.y, b = blockIdx.z % p.B, split = blockIdx.z / p.B;
    const int h_begin = first_head(p, split), g = first_head(p, split + 1) - h_begin, rows = p.N * g;
    const GlobalMask mask = global_mask(p, b);
    load_transposed<T, DP, BM>(kt, p.d, p.vec, [&](int r) -> const T * { return j0 + r < mask.len ? at<T>(p.k, p.ks, b, j0 + r, kh) : nullptr; });
    load_transposed<T, DP, BM>(vt, p.d, p.vec, [&](int r) -> const T * { return j0 + r < mask.len ? at<T>(p.v, p.vs, b, j0 + r, kh) : nullptr; });
    float acc_k[RM][NC] = {}, acc_v[RM][NC] = {};
    float2 here[RM];
    int doc_of[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int j = j0 + RM * ty + i;
        here[i] = map_place(j, p.width);
        doc_of[i] = p.k_docs && j < p.M ? p.k_docs[static_cast<long long>(b) * p.M + j] : p.k_docs ? -1 : 0;
    }
    if (p.k_docs) {
        if (tid == 0) range[0] = 0x7fffffff, range[1] = -1;
        __syncthreads();
        if (tx == 0) {
#pragma unroll
            for (int i = 0; i < RM; ++i)
                if (doc_of[i] >= 0) {
                    atomicMin(range, doc_of[i]);
                    atomicMax(range + 1, doc_of[i]);
                }
        }
        __syncthreads();
    }
    const long long first = static_cast<long long>(query_begin(mask, j0)) * g;
    Tile<T, DP, BN> tile;
    const auto fetch_q = [&](int r0) {
        tile.fetch(p.d, p.vec, [&](int r) -> const T * {
            if (r0 + r >= rows) return nullptr;
            const RowOf t = row_of(p, kh, r0 + r, g, h_begin);
            return at<T>(p.q, p.qs, b, t.n, t.head);
        });
    };
    const int r_begin = first < rows ? static_cast<int>(first) / BN * BN : rows;
    if (!p.q_docs && r_begin < rows) fetch_q(r_begin);
    for (int r0 = r_begin; r0 < rows; r0 += BN) {
        __syncthreads();
        bool any = true;
        if (tid < BN) {
            const bool in = r0 + tid < rows;
            const RowOf t = row_of(p, kh, min(r0 + tid, rows - 1), g, h_begin);
            const long long row = (static_cast<long long>(b) * p.h + t.head) * p.N + t.n;
            place[tid] = map_place(t.n + mask.shift, p.width);
            lse[tid] = p.lse[row];
            delta[tid] = p.delta[row];
            slope[tid] = p.slopes ? p.slopes[t.head] * kLog2e : 0.0f;
            n_of[tid] = in ? t.n : -1;
            if (p.q_docs) {
                const int dq = in ? p.q_docs[static_cast<long long>(b) * p.N + t.n] : -1;
                doc[tid] = dq;
                any = dq >= range[0] && dq <= range[1];
            }
        } else if (p.q_docs) {
            any = false;
        }
        if (p.q_docs) {
            if (!__syncthreads_or(any)) continue;
            fetch_q(r0);
        }
        const bool odd_q = tile.put(qot);
        __syncthreads();
        tile.fetch(p.d, p.vec, [&](int r) -> const T * {
            if (r0 + r >= rows) return nullptr;
            const RowOf t = row_of(p, kh, r0 + r, g, h_begin);
            return static_cast<const T *>(p.d_out) + ((static_cast<long long>(b) * p.N + t.n) * p.h + t.head) * p.d;
        });
        float s[RM][RN] = {}, dp[RM][RN] = {};
        products<RM, RN, PM, PN>(s, kt, qot, p.d, ty, tx);
        __syncthreads();
        const bool odd_o = tile.put(qot);
        const bool bad = __syncthreads_or(odd_q || odd_o);
        fetch_q(r0);
        products<RM, RN, PM, PN>(dp, vt, qot, p.d, ty, tx);
        if (p.cap != 0.0f) capped(s, p.scale / p.cap);
        const float unit = (p.cap != 0.0f ? p.cap : p.scale) * kLog2e;
        // (queries that stand before all of the tile's keys, or behind the last row, need the masks)
        const bool whole = !p.q_docs && r0 + BN <= rows && j0 + BM <= key_end(mask, r0 / g);
        const auto seen = [&](int i, int c) {
            const int id = p.k_docs ? doc[c] : 0, n = n_of[c];
            return n >= 0 && sees(mask, n, j0 + RM * ty + i) && id == doc_of[i] && id >= 0;
        };
#pragma unroll
        for (int j = 0; j < RN; ++j) {
            const int c = RN * tx + j;
            const float less = delta[c], level = lse[c];
#pragma unroll
            for (int i = 0; i < RM; ++i) {
                dp[i][j] -= less;
                if (p.cap != 0.0f) dp[i][j] *= fmaf(-s[i][j], s[i][j], 1.0f);
                s[i][j] = fmaf(s[i][j], unit, -level);
            }
        }
        if (p.slopes) {
#pragma unroll
            for (int j = 0; j < RN; ++j) {
                const float2 there = place[RN * tx + j];
                const float steep = slope[RN * tx + j];
#pragma unroll
                for (int i = 0; i < RM; ++i) s[i][j] -= steep * map_distance(here[i], there);
            }
        }
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < RN; ++j) {
                s[i][j] = exp2_fast(s[i][j]);
                dp[i][j] *= s[i][j];
            }
        if (!whole) {
#pragma unroll
            for (int j = 0; j < RN; ++j) {
                const int c = RN * tx + j, id = p.k_docs ? doc[c] : 0, n = n_of[c];
#pragma unroll
                for (int i = 0; i < RM; ++i)
                    if (n < 0 || !sees(mask, n, j0 + RM * ty + i) || id != doc_of[i] || id < 0) s[i][j] = dp[i][j] = 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < RN; ++j) w[(RM * ty + i) * PN + RN * tx + j] = s[i][j];
        __syncthreads();
        accumulate<RM, NC, BN>(acc_v, w, qot, ty, tx, bad, seen);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < RN; ++j) w[(RM * ty + i) * PN + RN * tx + j] = dp[i][j];
        tile.put(qot);
        __syncthreads();
        if (!p.q_docs && r0 + BN < rows) fetch_q(r0 + BN);
        accumulate<RM, NC, BN>(acc_k, w, qot, ty, tx, bad, seen);
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int j = j0 + RM * ty + i;
        if (j >= p.M) continue;
        const long long o = ((static_cast<long long>(b) * p.M + j) * p.hk + kh) * p.d;
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if (tx + 16 * c < p.d) {
                if (p.head_splits > 1) {
                    const long long part = static_cast<long long>(split) * p.B * p.M * p.hk * p.d + o + tx + 16 * c;
                    p.part_k[part] = acc_k[i][c] * p.scale;
                    p.part_v[part] = acc_v[i][c];
                } else {
                    store_one<T>(static_cast<T *>(p.d_k) + o + tx + 16 * c, acc_k[i][c] * p.scale);
                    store_one<T>(static_cast<T *>(p.d_v) + o + tx + 16 * c, acc_v[i][c]);
                }
            }
    }
}

template <typename... A>
cudaError_t launch_any(void (*kernel)(GlobalParams), dim3 grid, size_t smem, cudaStream_t stream, const GlobalParams &p)
{
    // per device and cheap; more than 48 KB needs the attribute
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (err != cudaSuccess) return err;
    return launch_chained(kernel, grid, kAnyThreads, smem, stream, p);
}

template <typename T, int DP, int RM, int RN>
cudaError_t forward_one(const GlobalParams &p, cudaStream_t stream)
{
    constexpr int BM = 16 * RM, BN = 16 * RN;
    constexpr size_t smem = sizeof(float) * (DP * (BM + 4) + DP * (BN + 4) + BM * (BN + 4) + 2 * BN + BN + 2);
    static_assert(smem <= 227 * 1024, "shared memory of a block");
    const dim3 grid((p.N * p.g + BM - 1) / BM, p.hk, p.B * p.splits);
    return launch_any(global_any_forward_kernel<T, DP, RM, RN>, grid, smem, stream, p);
}

// Blocks of 128 rows, eight per thread, read shared memory half as often per multiplication as blocks of 64; they pay once they
// fill the chip.
bool any_fills(const GlobalParams &p, int rows, int block, int splits = 1)
{
    return 1LL * ((rows + block - 1) / block) * p.hk * p.B * splits >= sm_count() * 3 / 4;
}

template <typename T, int DP>
cudaError_t forward_width(const GlobalParams &p, cudaStream_t stream)
{
    // sixteen rows or fewer (single tokens): a block of sixteen rows
    if (p.N * p.g <= 16) return forward_one<T, DP, 1, 4>(p, stream);
    if constexpr (DP > 128) return forward_one<T, DP, 2, 2>(p, stream);
    else return any_fills(p, p.N * p.g, 128) && p.splits == 1 ? forward_one<T, DP, 8, 4>(p, stream) : forward_one<T, DP, 4, 4>(p, stream);
}

template <int DP, int RM, int RN>
constexpr size_t backward_shared()
{
    constexpr int BM = 16 * RM, BN = 16 * RN;
    constexpr size_t smem = sizeof(float) * (2 * DP * (BM + 4) + DP * (BN + 4) + BM * (BN + 4) + 7 * BN + 2);
    static_assert(smem <= 227 * 1024, "shared memory of a block");
    return smem;
}

template <typename T, int DP, int RM, int RN>
cudaError_t dq_one(const GlobalParams &p, cudaStream_t stream)
{
    return launch_any(global_any_dq_kernel<T, DP, RM, RN>, dim3((p.N * p.g + 16 * RM - 1) / (16 * RM), p.hk, p.B), backward_shared<DP, RM, RN>(), stream, p);
}

template <typename T, int DP, int RM, int RN>
cudaError_t dkv_one(const GlobalParams &p, cudaStream_t stream)
{
    return launch_any(global_any_dkv_kernel<T, DP, RM, RN>, dim3((p.M + 16 * RM - 1) / (16 * RM), p.hk, p.B * p.head_splits), backward_shared<DP, RM, RN>(), stream, p);
}

// Each pass has the largest blocks that fill the chip: 128 rows, 64 or 32.
template <typename T, int DP>
cudaError_t backward_width(const GlobalParams &p, cudaStream_t stream)
{
    if constexpr (DP > 128) {
        const cudaError_t err = dq_one<T, DP, 2, 2>(p, stream);
        return err != cudaSuccess ? err : dkv_one<T, DP, 2, 2>(p, stream);
    } else {
        const cudaError_t err = any_fills(p, p.N * p.g, 128)  ? dq_one<T, DP, 8, 4>(p, stream)
                                : any_fills(p, p.N * p.g, 64) ? dq_one<T, DP, 4, 4>(p, stream)
                                                              : dq_one<T, DP, 2, 4>(p, stream);
        if (err != cudaSuccess) return err;
        return any_fills(p, p.M, 128, p.head_splits)  ? dkv_one<T, DP, 8, 4>(p, stream)
               : any_fills(p, p.M, 64, p.head_splits) ? dkv_one<T, DP, 4, 4>(p, stream)
                                                      : dkv_one<T, DP, 2, 4>(p, stream);
    }
}

template <typename T>
cudaError_t any_type(const GlobalParams &p, bool back, cudaStream_t stream)
{
    if (p.d <= 32) return back ? backward_width<T, 32>(p, stream) : forward_width<T, 32>(p, stream);
    if (p.d <= 64) return back ? backward_width<T, 64>(p, stream) : forward_width<T, 64>(p, stream);
    if (p.d <= 128) return back ? backward_width<T, 128>(p, stream) : forward_width<T, 128>(p, stream);
    return back ? backward_width<T, 256>(p, stream) : forward_width<T, 256>(p, stream);
}

}  // namespace

cudaError_t run_global_any_forward(const GlobalParams &p, int dtype, cudaStream_t stream)
{
    switch (dtype) {
    case MATCHATTN_F32: return any_type<float>(p, false, stream);
    case MATCHATTN_F16: return any_type<__half>(p, false, stream);
    default: return any_type<__nv_bfloat16>(p, false, stream);
    }
}

cudaError_t run_global_any_backward(const GlobalParams &p, int dtype, cudaStream_t stream)
{
    switch (dtype) {
    case MATCHATTN_F32: return any_type<float>(p, true, stream);
    case MATCHATTN_F16: return any_type<__half>(p, true, stream);
    default: return any_type<__nv_bfloat16>(p, true, stream);
    }
}

}  // namespace matchattn
