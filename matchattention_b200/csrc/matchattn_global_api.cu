// Dense attention: entry points, the choice of kernels, and the small kernels around them.
#include "matchattn_global_mma.cuh"

namespace matchattn {
namespace {

// out = sum over the splits of 2^(lse_s - lse) * part_s: a warp per row of a head.  Reads the parts once (float32), bound by
// their latency: 256 rows of ten shares 9 us with a branch between a share's figure and its part.  At most 64 shares.
template <typename T>
__global__ void __launch_bounds__(256) global_join_kernel(const GlobalParams p)
{
    chain_begin();
    const long long rows = static_cast<long long>(p.B) * p.h * p.N;
    const long long row = blockIdx.x * 8LL + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int lane = threadIdx.x & 31;
    // a lane has the figures of up to two shares; one that holds no key that the row sees has minus infinity, and zeros
    float x[2], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        x[i] = lane + 32 * i < p.splits ? p.part_lse[(lane + 32 * i) * rows + row] : -INFINITY;
        top = fmaxf(top, x[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float ref = top == -INFINITY ? 0.0f : top;
    x[0] = exp2f(x[0] - ref), x[1] = exp2f(x[1] - ref);
    float sum = x[0] + x[1], acc[8] = {};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        const float w = __shfl_sync(0xffffffffu, s < 32 ? x[0] : x[1], s & 31);
        const float *part = p.part_out + (s * rows + row) * p.d;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < p.d) acc[i] = fmaf(w, part[lane + 32 * i], acc[i]);
    }
    const int n = static_cast<int>(row % p.N);
    const long long bh = row / p.N, b = bh / p.h, head = bh - b * p.h;
    const bool empty = sum == 0.0f;
    if (p.lse && lane == 0) p.lse[row] = empty ? INFINITY : ref + log2f(sum);
    const long long out = ((b * p.N + n) * p.h + head) * p.d;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < p.d) store_result<T>(p, out + lane + 32 * i, empty ? 0.0f : acc[i] / sum);
}

// A sum over the channels of V per lane, `lanes` to a row.
template <typename T, int V>
__device__ __forceinline__ void read_channels(const T *p, float (&x)[V])
{
    if constexpr (V == 1) {
        x[0] = load_one<T>(p);
    } else {
        const uint4 t = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = DT<T>::unpack(w[i / DT<T>::kElemsPerWord], i % DT<T>::kElemsPerWord);
    }
}

// delta = sum over the channels of d_out * out (with what its rounding left): `lanes` lanes per row, V channels at a time (16 bytes, or
// one element).  Bound by memory; 2 x 4096 tokens, 16 heads x 128, bfloat16, by single elements and a warp per row 36 us.
template <typename T, int V>
__global__ void __launch_bounds__(256) global_delta_kernel(const GlobalParams p, int lanes)
{
    chain_begin();
    const long long rows = static_cast<long long>(p.B) * p.N * p.h;
    const long long row = static_cast<long long>(blockIdx.x) * (256 / lanes) + threadIdx.x / lanes;
    const int lane = threadIdx.x & (lanes - 1);
    float sum = 0.0f;
    if (row < rows) {
        const T *o = static_cast<const T *>(p.out) + row * p.d, *g = static_cast<const T *>(p.d_out) + row * p.d;
        const T *low = p.low ? static_cast<const T *>(p.low) + row * p.d : nullptr;
        for (int c = lane * V; c < p.d; c += lanes * V) {
            float x[V], y[V], z[V] = {};
            read_channels<T, V>(o + c, x);
            read_channels<T, V>(g + c, y);
            if (low) read_channels<T, V>(low + c, z);
#pragma unroll
            for (int i = 0; i < V; ++i) sum = fmaf(x[i], y[i], fmaf(z[i], y[i], sum));
        }
    }
    for (int i = lanes / 2; i > 0; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
    if (row < rows && lane == 0) {
        const long long bn = row / p.h, head = row - bn * p.h, b = bn / p.N, n = bn - b * p.N;
        p.delta[(b * p.h + head) * p.N + n] = sum;
    }
}

template <typename T>
cudaError_t find_delta(const GlobalParams &p, bool wide, cudaStream_t stream)
{
    constexpr int V = 16 / sizeof(T);
    int lanes = 32;
    while (wide && lanes > 1 && lanes / 2 * V >= p.d) lanes /= 2;
    const long long rows = 1LL * p.B * p.N * p.h;
    const dim3 grid(static_cast<unsigned>((rows + 256 / lanes - 1) / (256 / lanes)));
    return wide ? launch_chained(global_delta_kernel<T, V>, grid, 256, 0, stream, p, lanes)
                : launch_chained(global_delta_kernel<T, 1>, grid, 256, 0, stream, p, lanes);
}

// Whether some query sees key j of item b.  Without documents the last query sees every key there is.
__device__ __forceinline__ bool key_seen(const GlobalParams &p, const GlobalMask &mask, int b, int j, int query_tiles)
{
    if (j >= mask.len) return false;
    if (p.k_docs == nullptr) return true;
    const int id = p.k_docs[static_cast<long long>(b) * p.M + j], first = query_begin(mask, j), own = j - mask.shift;
    if (id < 0) return false;
    const int *ids = p.q_docs + static_cast<long long>(b) * p.N;
    // (mostly the query that stands at the key)
    if (own >= first && own < p.N && ids[own] == id) return true;
    for (int t = first / kTile; t < query_tiles; ++t) {
        const DocRange r = p.ranges[b * query_tiles + t];
        if (id < r.low || id > r.high) continue;
        for (int n = max(first, t * kTile); n < min((t + 1) * kTile, p.N); ++n)
            if (ids[n] == id) return true;
    }
    return false;
}

// float16: what bounds dS, per tile of 128 tokens of a head (level_o, level_delta, level_v): blocks of query tiles, then of key tiles, two
// lanes to a row.  Only tokens that take part in a visible pair count (what is hidden has no say in how the rest is held), and of those only
// finite figures: infinities and NaN reach the results whatever they are held by.  Bound by memory.
__global__ void __launch_bounds__(2 * kTile) global_levels_kernel(const GlobalParams p)
{
    chain_begin();
    const int query_tiles = (p.N + kTile - 1) / kTile, key_tiles = (p.M + kTile - 1) / kTile, query_blocks = p.B * p.h * query_tiles;
    const bool keys = static_cast<int>(blockIdx.x) >= query_blocks;
    const int i = keys ? blockIdx.x - query_blocks : blockIdx.x, tiles = keys ? key_tiles : query_tiles, heads = keys ? p.hk : p.h;
    const int bh = i / tiles, row = (i - bh * tiles) * kTile + threadIdx.x / 2, b = bh / heads, head = bh - b * heads;
    const __half *x = nullptr;
    float square = 0.0f, delta = 0.0f;
    if (keys) {
        if (key_seen(p, global_mask(p, b), b, row, query_tiles)) x = static_cast<const __half *>(p.v) + b * p.vs[0] + row * p.vs[1] + head * p.vs[2];
    } else if (row < p.N) {
        const long long line = static_cast<long long>(bh) * p.N + row;
        // (a query that sees nothing has an infinite lse)
        if (p.lse[line] != INFINITY) {
            x = static_cast<const __half *>(p.d_out) + ((static_cast<long long>(b) * p.N + row) * p.h + head) * p.d;
            delta = fabsf(p.delta[line]);
        }
    }
    if (x != nullptr)
        for (int c = threadIdx.x % 2 * 8; c < p.d; c += 16) {
            float y[8];
            read_channels<__half, 8>(x + c, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) square = fmaf(y[e], y[e], square);
        }
    square += __shfl_xor_sync(0xffffffffu, square, 1);
    float norm = sqrtf(square);
    norm = norm <= 3.402823466e38f ? norm : 0.0f;
    delta = delta <= 3.402823466e38f ? delta : 0.0f;
    for (int o = 16; o > 1; o >>= 1) {
        norm = fmaxf(norm, __shfl_xor_sync(0xffffffffu, norm, o));
        delta = fmaxf(delta, __shfl_xor_sync(0xffffffffu, delta, o));
    }
    __shared__ float most[2][kTile / 16];
    if (threadIdx.x % 32 == 0) most[0][threadIdx.x / 32] = norm, most[1][threadIdx.x / 32] = delta;
    __syncthreads();
    if (threadIdx.x < 2) {
        float level = 0.0f;
        for (int w = 0; w < kTile / 16; ++w) level = fmaxf(level, most[threadIdx.x][w]);
        if (keys && threadIdx.x == 0) p.level_v[i] = level;
        if (!keys) (threadIdx.x == 0 ? p.level_o : p.level_delta)[i] = level;
    }
}

// dK and dV as the sums of their parts over the blocks that shared out the query heads, four elements per thread (one at the end).
template <typename T>
__global__ void __launch_bounds__(256) global_join_heads_kernel(const GlobalParams p)
{
    chain_begin();
    const long long n = static_cast<long long>(p.B) * p.M * p.hk * p.d, i0 = (blockIdx.x * 256LL + threadIdx.x) * 4;
    const float *part = blockIdx.y ? p.part_v : p.part_k;
    T *to = static_cast<T *>(blockIdx.y ? p.d_v : p.d_k);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (i0 + e >= n) return;
        float sum = 0.0f;
        for (int s = 0; s < p.head_splits; ++s) sum += part[s * n + i0 + e];
        store_one<T>(to + i0 + e, sum);
    }
}

// What the ids of a block of 128 tokens span: blocks of queries of all items, then blocks of keys.
__global__ void __launch_bounds__(kTile) global_ranges_kernel(const GlobalParams p, DocRange *ranges)
{
    chain_begin();
    const int query_tiles = (p.N + kTile - 1) / kTile, key_tiles = (p.M + kTile - 1) / kTile;
    const bool keys = blockIdx.x >= p.B * query_tiles;
    const int i = keys ? blockIdx.x - p.B * query_tiles : blockIdx.x, tiles = keys ? key_tiles : query_tiles, rows = keys ? p.M : p.N;
    const int b = i / tiles, row = (i - b * tiles) * kTile + threadIdx.x;
    const bool in = row < rows;
    const int id = in ? (keys ? p.k_docs : p.q_docs)[static_cast<long long>(b) * rows + row] : -1;
    __shared__ int low, high, impure;
    if (threadIdx.x == 0) low = 0x7fffffff, high = -1, impure = 0;
    __syncthreads();
    if (in && id < 0) impure = 1;
    if (in && id >= 0) {
        atomicMin(&low, id);
        atomicMax(&high, id);
    }
    __syncthreads();
    if (threadIdx.x == 0) ranges[blockIdx.x] = DocRange{low, high, !impure, 0};
}

template <typename F>
cudaError_t by_type(int dtype, F f)
{
    switch (dtype) {
    case MATCHATTN_F32: return f(float());
    case MATCHATTN_F16: return f(__half());
    default: return f(__nv_bfloat16());
    }
}

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_global(const matchattn_global_args *a)
{
    if (a == nullptr || !a->q || !a->out || (a->M > 0 && (!a->k || !a->v))) return MATCHATTN_ERR_NULL;
    if ((a->q_docs == nullptr) != (a->k_docs == nullptr)) return MATCHATTN_ERR_NULL;
    if (a->B <= 0 || a->N <= 0 || a->M < 0 || a->h <= 0 || a->hk <= 0 || a->h % a->hk != 0 || a->d <= 0 || a->d > MATCHATTN_MAX_DENSE_D ||
        a->width <= 0)
        return MATCHATTN_ERR_SHAPE;
    // The kernels work with scale, cap and their quotient in units of log2: what these make infinite, zero or less than a normal number would
    // give NaN, or another function.  (Written so that NaN fails.)
    constexpr float least = 1.175494351e-38f, most = 3.402823466e38f / kLog2e;
    if (!(a->scale >= least && a->scale <= most)) return MATCHATTN_ERR_SHAPE;
    if (a->cap != 0.0f && !(a->cap >= least && a->cap <= most && a->scale / a->cap >= least && a->scale / a->cap <= most)) return MATCHATTN_ERR_SHAPE;
    if (a->prefix && !a->causal) return MATCHATTN_ERR_SHAPE;
    if (a->dtype < MATCHATTN_F32 || a->dtype > MATCHATTN_BF16) return MATCHATTN_ERR_DTYPE;
    const size_t size = a->dtype == MATCHATTN_F32 ? 4 : 2;
    if (!aligned(a->q, size) || !aligned(a->k, size) || !aligned(a->v, size) || !aligned(a->out, size) || !aligned(a->out_low, size) || !aligned(a->lse, 4) ||
        !aligned(a->slopes, 4) || !aligned(a->prefix, 4) || !aligned(a->lengths, 4) || !aligned(a->q_docs, 4) || !aligned(a->k_docs, 4))
        return MATCHATTN_ERR_ALIGN;
    // positions are exact in float32; rows of a key head and grid dimensions are 32- and 16-bit
    if (a->N > (1 << 24) || a->M > (1 << 24) || a->h > 65535 || a->B > 65535 || 1LL * a->N * (a->h / a->hk) > (1LL << 30) ||
        1LL * a->B * a->h * (a->N / kTile + 1) > (1LL << 26) || 1LL * a->B * a->hk * (a->M / kTile + 1) > (1LL << 26))
        return MATCHATTN_ERR_TOO_LARGE;
    return MATCHATTN_OK;
}

// Shares of the keys of a forward call with few blocks: enough to fill the SMs, none shorter than four tiles.
int splits_of(long long blocks, int tiles, int B)
{
    const long long fill = sm_count();
    if (blocks >= fill / 2 || tiles < 8) return 1;
    long long s = (2 * fill) / blocks;
    if (s > tiles / 4) s = tiles / 4;
    if (s > 64) s = 64;
    while (s > 1 && s * B > 65535) --s;
    return s < 2 ? 1 : static_cast<int>(s);
}

// Queries times sharing heads up to which a call counts as one of single tokens: the rows of a warp's matrix instruction.
constexpr int kTokenRows = 16;

// Keys from which the matrix kernel holds float16 probabilities by more (matchattn_global_fwd.inl).  What a key's weight loses to rounding
// is 2^-33 of the largest at most, of so many keys 2^-17: a thirty-second of a half step of the type, against the largest value.
constexpr int kManyKeys = 1 << 16;

bool matrix_call(const matchattn_global_args *a)
{
    return a->dtype != MATCHATTN_F32 && a->d <= 128 && a->d % 8 == 0 && aligned(a->out, 16) && aligned(a->out_low, 16) && rows_fit(a->q, a->q_stride, a->B, a->N, a->h) &&
           rows_fit(a->k, a->k_stride, a->B, a->M, a->hk) && rows_fit(a->v, a->v_stride, a->B, a->M, a->hk);
}

struct Plan {
    bool matrix, token;
    int block_rows, splits, tiles_per_split;
    size_t part_out, part_lse;      // floats
    size_t ranges;                  // DocRange
    size_t bytes() const { return ranges * sizeof(DocRange) + sizeof(float) * (part_out + part_lse); }
};

size_t range_count(const matchattn_global_args *a)
{
    return a->q_docs ? static_cast<size_t>(a->B) * ((a->N + kTile - 1) / kTile + (a->M + kTile - 1) / kTile) : 0;
}

Plan plan_forward(const matchattn_global_args *a)
{
    const int g = a->h / a->hk, rows = a->N * g;
    Plan p{};
    p.matrix = rows > kTokenRows && matrix_call(a);
    p.token = rows <= kTokenRows && matrix_call(a);
    int tiles;
    long long blocks;
    if (p.token) {
        blocks = 1LL * a->hk * a->B;
        tiles = (a->M + kTile - 1) / kTile;
        // two blocks per SM, of eight runs of keys per warp at least.  8 items of 2048 to 8192 keys, 32 heads on 8 key heads x 128, bf16,
        // with the join: two blocks per SM 52 us, four 60, eight 69
        const long long most = tiles / 4, wanted = (2LL * sm_count() + blocks - 1) / blocks;
        p.splits = static_cast<int>(wanted < most ? wanted : most);
        if (p.splits > 64) p.splits = 64;
    } else if (p.matrix) {
        // two tiles of queries keep the matrix unit and the exponentials busy at once; one where two leave SMs idle
        blocks = 1LL * ((a->N + 2 * kTile - 1) / (2 * kTile)) * a->h * a->B;
        p.block_rows = 2 * kTile;
        if (blocks < sm_count()) {
            p.block_rows = kTile;
            blocks = 1LL * ((a->N + kTile - 1) / kTile) * a->h * a->B;
        }
        tiles = (a->M + kTile - 1) / kTile;
        p.ranges = range_count(a);
    } else {
        const int bm = any_forward_rows(rows, a->d), bn = any_forward_keys(rows, a->d);
        blocks = 1LL * ((rows + bm - 1) / bm) * a->hk * a->B;
        tiles = (a->M + bn - 1) / bn;
    }
    if (!p.token) p.splits = splits_of(blocks, tiles, a->B);
    if (p.splits < 1) p.splits = 1;
    p.tiles_per_split = p.splits > 1 ? (tiles + p.splits - 1) / p.splits : tiles;
    if (p.splits > 1) {
        p.splits = (tiles + p.tiles_per_split - 1) / p.tiles_per_split;
        p.part_lse = static_cast<size_t>(p.splits) * a->B * a->h * a->N;
        p.part_out = p.part_lse * a->d;
    }
    return p;
}

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                              const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's tensor-map encoder, looked up through the runtime (the library does not link libcuda).
EncodeFn encoder()
{
    static const EncodeFn fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        if (status_of(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q)) != MATCHATTN_OK || q != cudaDriverEntryPointSuccess)
            return static_cast<EncodeFn>(nullptr);
        return reinterpret_cast<EncodeFn>(f);
    }();
    return fn;
}

// Dimensions without a second element have a stride that nothing uses: one that the encoder accepts.
cudaError_t tile_map(CUtensorMap *map, const void *base, const long long (&stride)[3], int B, int rows, int heads, int d, int dtype)
{
    const EncodeFn encode = encoder();
    if (encode == nullptr) return cudaErrorNotSupported;
    const auto bytes = [](long long s, int size) { return static_cast<cuuint64_t>(size > 1 ? 2 * s : 16); };
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(B)};
    const cuuint64_t strides[3] = {bytes(stride[2], heads), bytes(stride[1], rows), bytes(stride[0], B)};
    const cuuint32_t box[4] = {64, 1, kTile, 1}, each[4] = {1, 1, 1, 1};
    const CUresult r = encode(map, dtype == MATCHATTN_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base),
                              dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

cudaError_t operand_maps(GlobalMaps &maps, const matchattn_global_args *a)
{
    cudaError_t err = tile_map(&maps.q, a->q, a->q_stride, a->B, a->N, a->h, a->d, a->dtype);
    if (err == cudaSuccess) err = tile_map(&maps.k, a->k, a->k_stride, a->B, a->M, a->hk, a->d, a->dtype);
    if (err == cudaSuccess) err = tile_map(&maps.v, a->v, a->v_stride, a->B, a->M, a->hk, a->d, a->dtype);
    return err;
}

cudaError_t find_ranges(GlobalParams &p, DocRange *ranges, cudaStream_t stream)
{
    if (p.q_docs == nullptr) return cudaSuccess;
    p.ranges = ranges;
    const unsigned blocks = static_cast<unsigned>(p.B) * ((p.N + kTile - 1) / kTile + (p.M + kTile - 1) / kTile);
    return launch_chained(global_ranges_kernel, dim3(blocks), kTile, 0, stream, p, ranges);
}

GlobalParams params_of(const matchattn_global_args *a)
{
    GlobalParams p{};
    p.q = a->q, p.k = a->k, p.v = a->v, p.out = a->out, p.lse = a->lse;
    p.low = a->dtype == MATCHATTN_F32 ? nullptr : a->out_low;
    for (int i = 0; i < 3; ++i) p.qs[i] = a->q_stride[i], p.ks[i] = a->k_stride[i], p.vs[i] = a->v_stride[i];
    p.slopes = a->slopes, p.prefix = a->prefix, p.lengths = a->lengths, p.q_docs = a->q_docs, p.k_docs = a->k_docs;
    p.B = a->B, p.N = a->N, p.M = a->M, p.h = a->h, p.hk = a->hk, p.g = a->h / a->hk, p.d = a->d;
    p.causal = a->causal != 0, p.width = a->width, p.scale = a->scale, p.cap = a->cap;
    p.splits = p.head_splits = 1;
    const size_t run = 4 * (a->dtype == MATCHATTN_F32 ? 4 : 2);
    bool vec = a->d % 4 == 0 && aligned(a->q, run) && aligned(a->k, run) && aligned(a->v, run);
    for (int i = 0; i < 3; ++i) vec = vec && a->q_stride[i] % 4 == 0 && a->k_stride[i] % 4 == 0 && a->v_stride[i] % 4 == 0;
    p.vec = vec;
    return p;
}

// Scratch of the backward call: the documents of the tiles, parts of dK and dV, delta, in float16 the levels of the tiles.
size_t backward_floats(const matchattn_global_args *a) { return static_cast<size_t>(a->B) * a->h * a->N; }

// Blocks that share out the query heads of a key head in the pass for dK and dV, where its tiles of 128 keys leave SMs idle.
int head_splits(const matchattn_global_args *a)
{
    const int g = a->h / a->hk;
    const long long blocks = 1LL * ((a->M + kTile - 1) / kTile) * a->hk * a->B;
    if (g == 1 || blocks >= sm_count()) return 1;
    long long s = (sm_count() * 3LL / 2 + blocks - 1) / blocks;
    while (s > 1 && s * a->B > 65535) --s;
    return static_cast<int>(s < g ? s : g);
}

size_t part_floats(const matchattn_global_args *a)
{
    const int s = head_splits(a);
    return s > 1 ? static_cast<size_t>(s) * a->B * a->M * a->hk * a->d : 0;
}

// float16: of the query tiles twice, of the key tiles once
size_t query_levels(const matchattn_global_args *a) { return static_cast<size_t>(a->B) * a->h * ((a->N + kTile - 1) / kTile); }

size_t level_floats(const matchattn_global_args *a)
{
    return a->dtype == MATCHATTN_F16 ? 2 * query_levels(a) + static_cast<size_t>(a->B) * a->hk * ((a->M + kTile - 1) / kTile) : 0;
}

// (the parts come before delta, on 16 bytes)
size_t backward_bytes(const matchattn_global_args *a)
{
    return range_count(a) * sizeof(DocRange) + sizeof(float) * (2 * ((part_floats(a) + 3) / 4 * 4) + backward_floats(a) + level_floats(a));
}

}  // namespace
}  // namespace matchattn

using namespace matchattn;

extern "C" size_t matchattn_global_scratch_bytes(const matchattn_global_args *a, int backward)
{
    if (check_global(a) != MATCHATTN_OK || a->M == 0) return 0;
    if (backward) return backward_bytes(a);
    const Plan plan = plan_forward(a);
    return plan.bytes();
}

extern "C" int matchattn_global_forward(const matchattn_global_args *a, void *scratch, size_t scratch_bytes, void *cuda_stream)
{
    const int bad = check_global(a);
    if (bad != MATCHATTN_OK) return bad;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const size_t size = a->dtype == MATCHATTN_F32 ? 4 : 2;
    GlobalParams p = params_of(a);
    if (a->M == 0) {        // no key at all: zeros (lse, for the backward pass, is not read then)
        return status_of(cudaMemsetAsync(a->out, 0, static_cast<size_t>(a->B) * a->N * a->h * a->d * size, stream));
    }
    const Plan plan = plan_forward(a);
    p.splits = plan.splits, p.tiles_per_split = plan.tiles_per_split, p.block_rows = plan.block_rows;
    p.held = a->M < kManyKeys ? 7.0f : 11.0f;
    if (plan.bytes() != 0) {
        if (scratch == nullptr) return MATCHATTN_ERR_NULL;
        if (scratch_bytes < plan.bytes()) return MATCHATTN_ERR_SCRATCH_LIMIT;
        if (!aligned(scratch, 16)) return MATCHATTN_ERR_ALIGN;
        p.part_out = reinterpret_cast<float *>(static_cast<DocRange *>(scratch) + plan.ranges);
        p.part_lse = p.part_out + plan.part_out;
    }
    cudaError_t err;
    if (plan.matrix) {
        GlobalMaps maps{};
        err = operand_maps(maps, a);
        if (err == cudaSuccess) err = find_ranges(p, static_cast<DocRange *>(scratch), stream);
        if (err == cudaSuccess) err = a->dtype == MATCHATTN_F16 ? run_global_forward<__half>(p, maps, stream) : run_global_forward<__nv_bfloat16>(p, maps, stream);
    } else if (plan.token) {
        err = run_global_token(p, a->dtype, stream);
    } else {
        err = run_global_any_forward(p, a->dtype, stream);
    }
    if (err == cudaSuccess && plan.splits > 1) {
        const unsigned blocks = static_cast<unsigned>((plan.part_lse / plan.splits + 7) / 8);
        err = by_type(a->dtype, [&](auto t) { return launch_chained(global_join_kernel<decltype(t)>, dim3(blocks), 256, 0, stream, p); });
    }
    return status_of(err);
}

extern "C" int matchattn_global_backward(const matchattn_global_args *a, const void *d_out, void *d_q, void *d_k, void *d_v, void *scratch,
                                         size_t scratch_bytes, void *cuda_stream)
{
    const int bad = check_global(a);
    if (bad != MATCHATTN_OK) return bad;
    if (!d_out || !d_q || (a->M > 0 && (!d_k || !d_v || !a->lse || !scratch))) return MATCHATTN_ERR_NULL;
    const cudaStream_t stream = static_cast<cudaStream_t>(cuda_stream);
    const size_t size = a->dtype == MATCHATTN_F32 ? 4 : 2;
    if (!aligned(d_out, size) || !aligned(d_q, size) || !aligned(d_k, size) || !aligned(d_v, size)) return MATCHATTN_ERR_ALIGN;
    if (a->M == 0) return status_of(cudaMemsetAsync(d_q, 0, static_cast<size_t>(a->B) * a->N * a->h * a->d * size, stream));
    if (scratch_bytes < backward_bytes(a)) return MATCHATTN_ERR_SCRATCH_LIMIT;
    if (!aligned(scratch, 16)) return MATCHATTN_ERR_ALIGN;
    GlobalParams p = params_of(a);
    p.vec = p.vec && aligned(d_out, 4 * size);
    p.d_out = d_out, p.d_q = d_q, p.d_k = d_k, p.d_v = d_v;
    DocRange *ranges = static_cast<DocRange *>(scratch);
    p.head_splits = head_splits(a);
    p.part_k = reinterpret_cast<float *>(ranges + range_count(a));
    p.part_v = p.part_k + (part_floats(a) + 3) / 4 * 4;
    p.delta = p.part_v + (part_floats(a) + 3) / 4 * 4;
    const bool matrix = matrix_call(a) && aligned(d_out, 16) && aligned(d_q, 16) && aligned(d_k, 16) && aligned(d_v, 16);
    const bool wide = a->d % (16 / static_cast<int>(size)) == 0 && aligned(a->out, 16) && aligned(a->out_low, 16) && aligned(d_out, 16);
    cudaError_t err = by_type(a->dtype, [&](auto t) { return find_delta<decltype(t)>(p, wide, stream); });
    if (err == cudaSuccess && matrix) {
        GlobalMaps maps{};
        const long long stride[3] = {1LL * a->N * a->h * a->d, 1LL * a->h * a->d, a->d};
        err = operand_maps(maps, a);
        if (err == cudaSuccess) err = tile_map(&maps.o, d_out, stride, a->B, a->N, a->h, a->d, a->dtype);
        if (err == cudaSuccess) err = find_ranges(p, ranges, stream);
        if (err == cudaSuccess && a->dtype == MATCHATTN_F16) {
            p.level_o = p.delta + backward_floats(a);
            p.level_delta = p.level_o + query_levels(a);
            p.level_v = p.level_delta + query_levels(a);
            err = launch_chained(global_levels_kernel, dim3(static_cast<unsigned>(level_floats(a) - query_levels(a))), 2 * kTile, 0, stream, p);
        }
        if (err == cudaSuccess) err = a->dtype == MATCHATTN_F16 ? run_global_backward<__half>(p, maps, stream) : run_global_backward<__nv_bfloat16>(p, maps, stream);
    } else if (err == cudaSuccess) {
        err = run_global_any_backward(p, a->dtype, stream);
    }
    if (err == cudaSuccess && p.head_splits > 1) {
        const unsigned blocks = static_cast<unsigned>((static_cast<size_t>(a->B) * a->M * a->hk * a->d + 1023) / 1024);
        err = by_type(a->dtype, [&](auto t) { return launch_chained(global_join_heads_kernel<decltype(t)>, dim3(blocks, 2), 256, 0, stream, p); });
    }
    return status_of(err);
}
