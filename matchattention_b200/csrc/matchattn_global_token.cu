// Dense attention of few queries over many keys (new tokens over a cache), 16-bit types of up to 128 channels.
//
// The N x g query rows that share a key head, sixteen at most, are the sixteen rows of a warp's matrix instruction; a block of
// four warps takes a share of the keys of one key head, a warp every fourth run of sixteen keys.  Two blocks per SM: one begins or joins
// its parts while the other reads.  Bound by reading K and V
// once: the sixteen rows cost the instruction nothing more than one, and at 16 multiply-adds per value read it is idle most of the
// time (which is why the narrow warp-level instruction serves: nothing has to pass through shared or tensor memory).
//
// K and V go from global memory straight into the fragments, 16 bytes per load.  The order of the channels in a score's sum is free, so a
// lane's eight neighbouring channels are taken as its parts of two k-steps; the columns of the output are free too, so
// a lane's eight neighbouring channels of V are its column of eight column tiles (pairs of keys are put together by a byte
// permute).  The next run's keys are on their way while a run is computed.
//
// Measured, one B200: 8 items of 2048 to 8192 keys, 32 heads on 8 key heads x 128, bfloat16 47 us (DRAM at half its rate), the join 8; one item
// of 317 keys, 8 heads x 64, float16 4.9 us.  255 registers hold 8 KB per warp on their way, eight warps per SM: an SM with two full
// shares reads near its part of the memory's rate.  But the shares are cut from M, not from an item's own length: behind the shorter
// lengths blocks have nothing to read, and the longest share takes 1.4 to 1.7 times the mean.
//
// Each warp keeps its own maximum, sum and output; the warps are joined in shared memory, the shares of the keys by a second
// kernel.  Everything is float32 but the probabilities, which meet V as two terms of the type (rounded to it once they would make the largest
// error of a call: 2.2e-3 of the result in bfloat16 for 1.7e-3).  Up to eight rows the second terms are the other eight rows of the
// instruction, and cost nothing; beyond them they take a second one (32 heads on 8 key heads that way: 53 us for 50).  In float16 the
// probabilities and their sum are held times 2^15, the most that the type has room for: the many small weights of a long cache count.
#include "matchattn_global_mma.cuh"

namespace matchattn {
namespace {

constexpr int kTokenWarps = 4, kTokenThreads = 32 * kTokenWarps, kRun = 16;
template <typename T>
constexpr float kHeld = std::is_same<T, __half>::value ? 15.0f : 0.0f;

template <typename T>
__device__ __forceinline__ void warp_product(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x >= 0 in the type, rounded down, and what that left: not negative either, and for an x above 0 not zero, so that an infinite value meets
// two terms of one sign (2^-24 in float16, where x is up to 2^15)
template <typename T>
__device__ __forceinline__ float cut(float x)
{
    if constexpr (std::is_same<T, __half>::value) return __half2float(__float2half_rz(x));
    else return __uint_as_float(__float_as_uint(x) & 0xffff0000u);
}
template <typename T>
__device__ __forceinline__ float cut_off(float x)
{
    return x > 0.0f ? fmaxf(x - cut<T>(x), std::is_same<T, __half>::value ? 0x1p-24f : 0x1p-126f) : 0.0f;
}

__device__ __forceinline__ uint4 load_piece(const void *p, bool there)
{
    return there ? *static_cast<const uint4 *>(p) : make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ uint32_t word(const uint4 &x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

template <int DP>
struct TokenShared {
    float out[kTokenWarps][16][DP + 4];
    float top[kTokenWarps][16], sum[kTokenWarps][16];
    float prob[kTokenWarps][16][kRun];         // for runs that are added term by term
};

template <typename T, int DP>
__global__ void __launch_bounds__(kTokenThreads, 2) global_token_kernel(const GlobalParams p)
{
    chain_begin();
    constexpr int PIECES = DP / 32, GROUPS = DP / 64;
    extern __shared__ __align__(16) uint8_t raw_shared[];
    TokenShared<DP> &sh = *reinterpret_cast<TokenShared<DP> *>(raw_shared);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane >> 2, part = lane & 3;
    const int bk = blockIdx.x % (p.B * p.hk), split = blockIdx.x / (p.B * p.hk), b = bk / p.hk, kh = bk - b * p.hk;
    const int rows = p.N * p.g;
    const bool few = rows <= 8;                 // rows 8 to 15 of the instruction have the second terms of the probabilities
    const GlobalMask mask = global_mask(p, b);
    const T *keys = static_cast<const T *>(p.k) + b * p.ks[0] + kh * p.ks[2], *values = static_cast<const T *>(p.v) + b * p.vs[0] + kh * p.vs[2];
    const float factor = p.scale * kLog2e, inverse_cap = p.cap != 0.0f ? p.scale / p.cap : 0.0f, outer = p.cap * kLog2e;

    // rows quad and quad + 8 of the sixteen
    int limit[2], doc[2];
    float slope[2];
    float2 here[2];
    uint32_t query[PIECES][2][4];               // per piece of 32 channels: two k-steps of first operands
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = quad + 8 * i, n = min(r, rows - 1) / p.g, head = kh * p.g + min(r, rows - 1) - n * p.g;
        doc[i] = p.q_docs && r < rows ? p.q_docs[static_cast<long long>(b) * p.N + n] : 0;
        limit[i] = r < rows && doc[i] >= 0 ? key_limit(mask, n) : 0;
        slope[i] = p.slopes ? p.slopes[head] * kLog2e : 0.0f;
        here[i] = map_place(n + mask.shift, p.width);
        const T *q = static_cast<const T *>(p.q) + b * p.qs[0] + n * p.qs[1] + head * p.qs[2];
#pragma unroll
        for (int c = 0; c < PIECES; ++c) {
            const int at = 32 * c + 8 * part;
            const uint4 x = load_piece(q + at, r < rows && at < p.d);
            query[c][0][i] = x.x, query[c][0][2 + i] = x.y;
            query[c][1][i] = x.z, query[c][1][2 + i] = x.w;
        }
    }
    const int end = key_limit(mask, p.N - 1), all_see = key_limit(mask, 0);        // of the last and the first query
    const int j_begin = split * p.tiles_per_split * kTile;
    const int j_end = p.splits > 1 ? min(end, j_begin + p.tiles_per_split * kTile) : end;

    float out[GROUPS * 8][4] = {}, top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
    uint4 key[2][PIECES];
    const auto load_keys = [&](int j0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int j = j0 + 8 * i + quad;
            const T *row = keys + static_cast<long long>(min(j, p.M - 1)) * p.ks[1];
#pragma unroll
            for (int c = 0; c < PIECES; ++c) key[i][c] = load_piece(row + 32 * c + 8 * part, j < j_end && 32 * c + 8 * part < p.d);
        }
    };
    int j0 = j_begin + warp * kRun;
    if (j0 < j_end) load_keys(j0);
    for (; j0 < j_end; j0 += kTokenWarps * kRun) {
        // values of keys 2 part, 2 part + 1 and those eight further on
        uint4 value[GROUPS][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = j0 + 2 * part + (e & 1) + 8 * (e >> 1);
            const T *row = values + static_cast<long long>(min(j, p.M - 1)) * p.vs[1];
#pragma unroll
            for (int c = 0; c < GROUPS; ++c) value[c][e] = load_piece(row + 64 * c + 8 * quad, j < j_end && 64 * c + 8 * quad < p.d);
        }
        float s[2][4] = {};
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int c = 0; c < PIECES; ++c) {
                warp_product<T>(s[i], query[c][0], key[i][c].x, key[i][c].y);
                warp_product<T>(s[i], query[c][1], key[i][c].z, key[i][c].w);
            }
        load_keys(j0 + kTokenWarps * kRun);
        const bool partly = j0 + kRun > min(all_see, j_end) || p.k_docs != nullptr;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int j = j0 + 8 * i + 2 * part + e;
                const int id = p.k_docs && j < p.M ? p.k_docs[static_cast<long long>(b) * p.M + j] : 0;
                const float2 there = p.slopes ? map_place(j, p.width) : make_float2(0.0f, 0.0f);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float x = s[i][2 * r + e];
                    x = p.cap != 0.0f ? outer * tanh_one(x * inverse_cap) : x * factor;
                    if (p.slopes) x = fmaf(-slope[r], map_distance(here[r], there), x);
                    s[i][2 * r + e] = j < limit[r] && j < j_end && id == doc[r] ? x : -INFINITY;
                }
            }
        float base[2], shrink[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float high = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 1));
            high = fmaxf(fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 2)), top[r]);
            const float ref = high == -INFINITY ? 0.0f : high;
            shrink[r] = exp2_fast(top[r] - ref);
            base[r] = ref - kHeld<T>;
            top[r] = high;
            sum[r] *= shrink[r];
        }
        if (few) shrink[1] = shrink[0];
#pragma unroll
        for (int t = 0; t < GROUPS * 8; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) out[t][e] *= shrink[e / 2];
        uint32_t prob[4], rest[4];               // in two terms
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float e0 = exp2_fast(s[i][2 * r] - base[r]), e1 = exp2_fast(s[i][2 * r + 1] - base[r]);
                sum[r] += e0 + e1;
                prob[2 * i + r] = pack_two<T>(cut<T>(e0), cut<T>(e1));
                rest[2 * i + r] = pack_two<T>(cut_off<T>(e0), cut_off<T>(e1));
            }
        bool by_hand = false;
        if (partly) {
            uint32_t acc = 0;
#pragma unroll
            for (int c = 0; c < GROUPS; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc = taint<T>(value[c][e].x, taint<T>(value[c][e].y, taint<T>(value[c][e].z, taint<T>(value[c][e].w, acc))));
            by_hand = __any_sync(0xffffffffu, tainted<T>(acc));
        }
        const auto add = [&](auto both) {
#pragma unroll
            for (int c = 0; c < GROUPS; ++c)
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    const uint32_t pick = t & 1 ? 0x7632 : 0x5410;
                    const uint32_t low = __byte_perm(word(value[c][0], t / 2), word(value[c][1], t / 2), pick);
                    const uint32_t high = __byte_perm(word(value[c][2], t / 2), word(value[c][3], t / 2), pick);
                    warp_product<T>(out[8 * c + t], prob, low, high);
                    if constexpr (decltype(both)::value) warp_product<T>(out[8 * c + t], rest, low, high);
                }
        };
        if (!by_hand) {
            if (few) {
                prob[1] = rest[0], prob[3] = rest[2];
                add(std::false_type());
            } else {
                add(std::true_type());
            }
        } else {
            // values that are no numbers, and rows that do not see them: term by term, without the hidden terms (marked by -1)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int j = j0 + 8 * i + 2 * part + e;
                        const bool seen = j < limit[r] && j < j_end && (p.k_docs == nullptr || p.k_docs[static_cast<long long>(b) * p.M + j] == doc[r]);
                        sh.prob[warp][quad + 8 * r][8 * i + 2 * part + e] = seen ? DT<T>::unpack(prob[2 * i + r], e) + DT<T>::unpack(rest[2 * i + r], e) : -1.0f;
                    }
            __syncwarp();
            for (int e = 0; e < kRun && j0 + e < j_end; ++e) {
                const T *row = values + static_cast<long long>(j0 + e) * p.vs[1];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float x = sh.prob[warp][quad + 8 * r][e];
                    if (x < 0.0f) continue;
#pragma unroll
                    for (int t = 0; t < GROUPS * 8; ++t)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int c = t / 8 * 64 + 8 * (2 * part + u) + t % 8;
                            if (c < p.d) out[t][2 * r + u] = fmaf(x, load_one<T>(row + c), out[t][2 * r + u]);
                        }
                }
            }
            __syncwarp();
        }
    }
    if (few) {
#pragma unroll
        for (int t = 0; t < GROUPS * 8; ++t) out[t][0] += out[t][2], out[t][1] += out[t][3];
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
        if (part == 0) sh.top[warp][quad + 8 * r] = top[r], sh.sum[warp][quad + 8 * r] = sum[r];
#pragma unroll
        for (int c = 0; c < GROUPS; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float *to = &sh.out[warp][quad + 8 * r][64 * c + 8 * (2 * part + u)];
#pragma unroll
                for (int t = 0; t < 8; t += 4)
                    *reinterpret_cast<float4 *>(to + t) = make_float4(out[8 * c + t][2 * r + u], out[8 * c + t + 1][2 * r + u],
                                                                      out[8 * c + t + 2][2 * r + u], out[8 * c + t + 3][2 * r + u]);
            }
    }
    __syncthreads();
    // the warps' parts: a thread takes channel tid mod DP of every so many rows
    for (int i = tid; i < rows * DP; i += kTokenThreads) {
        const int r = i / DP, c = i % DP, n = r / p.g, head = kh * p.g + r - n * p.g;
        float high = -INFINITY;
#pragma unroll
        for (int w = 0; w < kTokenWarps; ++w) high = fmaxf(high, sh.top[w][r]);
        const float ref = high == -INFINITY ? 0.0f : high;
        float total = 0.0f, x = 0.0f;
#pragma unroll
        for (int w = 0; w < kTokenWarps; ++w) {
            // (a warp that has seen nothing of a row has zeros)
            const float weight = exp2_fast(sh.top[w][r] - ref);
            total = fmaf(weight, sh.sum[w][r], total);
            x = fmaf(weight, sh.out[w][r][c], x);
        }
        const bool empty = total == 0.0f;
        const long long line = (static_cast<long long>(b) * p.h + head) * p.N + n;
        const float result = empty ? 0.0f : x / total;
        if (p.splits > 1) {
            const long long at = static_cast<long long>(split) * p.B * p.h * p.N + line;
            if (c == 0) p.part_lse[at] = empty ? -INFINITY : ref + log2f(total) - kHeld<T>;
            if (c < p.d) p.part_out[at * p.d + c] = result;
        } else {
            if (c == 0 && p.lse) p.lse[line] = empty ? INFINITY : ref + log2f(total) - kHeld<T>;
            if (c < p.d) store_result<T>(p, ((static_cast<long long>(b) * p.N + n) * p.h + head) * p.d + c, result);
        }
    }
}

template <typename T, int DP>
cudaError_t token_one(const GlobalParams &p, cudaStream_t stream)
{
    const auto kernel = global_token_kernel<T, DP>;
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(TokenShared<DP>)));
    if (err != cudaSuccess) return err;
    return launch_chained(kernel, dim3(static_cast<unsigned>(p.B) * p.hk * p.splits), kTokenThreads, sizeof(TokenShared<DP>), stream, p);
}

}  // namespace

cudaError_t run_global_token(const GlobalParams &p, int dtype, cudaStream_t stream)
{
    if (dtype == MATCHATTN_F16) return p.d <= 64 ? token_one<__half, 64>(p, stream) : token_one<__half, 128>(p, stream);
    return p.d <= 64 ? token_one<__nv_bfloat16, 64>(p, stream) : token_one<__nv_bfloat16, 128>(p, stream);
}

}  // namespace matchattn
