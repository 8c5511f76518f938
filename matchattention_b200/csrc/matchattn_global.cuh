// Dense softmax attention over all keys that the masks leave (matchattn_global_forward, matchattn_global_backward): what its
// kernels share.
//
//   x_ij = scale * q_i.k_j;  with a cap: cap * tanh(x_ij / cap);  then  - slope_h * (|dx| + |dy|) of the two tokens
//   p_ij = exp(x_ij) / sum over the visible j,   out_i = sum_j p_ij v_j   (no visible key: zeros)
//
// Scores are kept in units of log2, so that a probability is one exp2.
#pragma once

#include "matchattn_kernels.cuh"

namespace matchattn {

constexpr float kLog2e = 1.4426950408889634f;

struct DocRange;

struct GlobalParams {
    const void *q, *k, *v;
    void *out, *low;         // [B, N, h, d]; low, 16-bit types: what the rounding of out left, or null
    float *lse;              // [B, h, N] log2 of the sum of 2^x of a row, +inf for a row that sees nothing; or null
    long long qs[3], ks[3], vs[3];      // strides in elements: item, token, head
    const float *slopes;                // [h] or null
    const int *prefix, *lengths;        // [B] or null
    const int *q_docs, *k_docs;         // [B, N], [B, M] or null
    int B, N, M, h, hk, g, d;           // g = h / hk query heads share a key head
    int causal, width;
    float scale, cap;                   // cap 0: none
    int vec;                            // rows of q, k and v can be read four elements at a time
    // forward with few queries: each split takes a share of the keys, a second kernel joins them
    int splits, tiles_per_split;
    int block_rows;                     // matrix kernels: queries of a block
    float held;                         // matrix kernels, float16: log2 of what probabilities are held by
    const DocRange *ranges;      // with documents: of the blocks of 128 queries, then of keys, item by item
    float *part_out, *part_lse;         // [splits, B, h, N, d], [splits, B, h, N]
    // backward
    const void *d_out;                  // [B, N, h, d]
    void *d_q, *d_k, *d_v;              // [B, N, h, d], [B, M, hk, d]
    float *delta;                       // [B, h, N] sum of d_out * out of a row
    int head_splits;                    // blocks of dK and dV that share out the query heads of a key head; their parts are joined after
    float *part_k, *part_v;             // [head_splits, B, M, hk, d]
    // float16, matrix kernels: per tile of 128 tokens of a head, the largest row norm of d_out and the largest delta, and of keys the largest
    // row norm of v
    float *level_o, *level_delta, *level_v;      // [B, h, query tiles] twice, [B, hk, key tiles]
};

// What an item's masks say.
struct GlobalMask {
    int len;        // keys [0, len) exist
    int shift;      // query n stands at key position n + shift
    int prefix;     // keys below it are seen whatever the causal order
    int causal;
};

__device__ __forceinline__ GlobalMask global_mask(const GlobalParams &p, int b)
{
    GlobalMask m;
    m.len = p.lengths ? min(max(p.lengths[b], 0), p.M) : p.M;
    m.shift = m.len - p.N;
    m.prefix = p.prefix ? p.prefix[b] : 0;
    m.causal = p.causal;
    return m;
}

__device__ __forceinline__ bool sees(const GlobalMask &m, int n, int j)
{
    return j < m.len && (!m.causal || j <= n + m.shift || j < m.prefix);
}

// Keys at and above this are seen by no query up to `n_last`.
__device__ __forceinline__ int key_end(const GlobalMask &m, int n_last)
{
    return m.causal ? min(m.len, max(max(n_last + m.shift + 1, m.prefix), 0)) : m.len;
}

// Queries below this see no key at or above `j_first`.
__device__ __forceinline__ int query_begin(const GlobalMask &m, int j_first)
{
    if (j_first >= m.len) return 1 << 30;
    return m.causal && j_first >= m.prefix ? max(0, j_first - m.shift) : 0;
}

// Column and row of a position on a map `width` tokens wide; positions before the first key are negative.
__device__ __forceinline__ float2 map_place(int pos, int width)
{
    int row = pos / width, col = pos - row * width;
    if (col < 0) {
        col += width;
        --row;
    }
    return make_float2(static_cast<float>(col), static_cast<float>(row));
}

__device__ __forceinline__ float map_distance(float2 a, float2 b) { return fabsf(a.x - b.x) + fabsf(a.y - b.y); }

// A result, and what its rounding left.
template <typename T>
__device__ __forceinline__ void store_result(const GlobalParams &p, long long at, float x)
{
    T *out = static_cast<T *>(p.out) + at;
    store_one<T>(out, x);
    if (sizeof(T) == 2 && p.low != nullptr) store_one<T>(static_cast<T *>(p.low) + at, x - DT<T>::rnd(x));
}

// Query heads (of the g that share a key head) of one of the blocks that share them out.
__device__ __forceinline__ int first_head(const GlobalParams &p, int split) { return split * p.g / p.head_splits; }

cudaError_t run_global_any_forward(const GlobalParams &p, int dtype, cudaStream_t stream);
cudaError_t run_global_any_backward(const GlobalParams &p, int dtype, cudaStream_t stream);

// Rows of a block and keys of a tile of the any-shape forward kernel: few query rows per key head take the low block.
constexpr int any_forward_rows(int rows, int d) { return d > 128 ? (rows <= 16 ? 16 : 32) : (rows <= 16 ? 16 : 64); }
constexpr int any_forward_keys(int rows, int d) { return d > 128 && rows > 16 ? 32 : 64; }

}  // namespace matchattn
