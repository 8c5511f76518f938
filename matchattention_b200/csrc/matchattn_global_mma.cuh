// Dense attention on the matrix units: tiles, barriers, tensor maps and the instructions around tcgen05.mma, for the kernels of
// matchattn_global_fwd.inl and matchattn_global_bwd.inl.
//
// Tiles.  128 rows (tokens) of a head, up to 128 channels, as one or two halves of 64 channels; a half is 128 rows of 128 bytes,
// 16-byte pieces swizzled by the row (piece ^ (row & 7)), as the tensor memory accelerator writes it and the matrix unit reads it.
// The same tile serves as an operand along its channels (scores) and along its rows (sums over the tokens).  Channels beyond d and
// rows beyond the tensor arrive as zeros.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "matchattn_global.cuh"

namespace matchattn {

constexpr int kTile = 128;                        // rows of a tile
constexpr int kHalfBytes = kTile * 128;           // 128 rows x 64 channels of 16 bits

struct GlobalMaps {
    CUtensorMap q, k, v, o;       // o: d_out (backward)
};

// lowest and highest id of a block of 128 tokens (ids that are not negative), and whether the block has no negative one
struct DocRange {
    int low, high, pure, unused;
};

// ---- shared-memory barriers ------------------------------------------------------------------------

__device__ __forceinline__ uint32_t shared_address(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void barrier_init(uint64_t *bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(bar)), "r"(count) : "memory");
}

__device__ __forceinline__ void barrier_expect(uint64_t *bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(bar)), "r"(bytes) : "memory");
}

__device__ __forceinline__ void barrier_arrive(uint64_t *bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_address(bar)) : "memory");
}

// One arrival for a whole warp, after all of it (a barrier serves the arrivals of 256 threads one by one, for a microsecond).
__device__ __forceinline__ void warp_arrive(uint64_t *bar)
{
    __syncwarp();
    if ((threadIdx.x & 31) == 0) barrier_arrive(bar);
}

__device__ __forceinline__ bool barrier_test(uint64_t *bar, uint32_t parity)
{
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(shared_address(bar)), "r"(parity)
                 : "memory");
    return done != 0;
}

__device__ __forceinline__ unsigned long long nanoseconds()
{
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// No wait of these kernels lasts longer than a tile's copies and products, microseconds; one of this length means that
// something is broken.  The block then raises its flag, every wait of it ends, and its results are NaN.
constexpr unsigned long long kWaitLimit = 2000000000ULL;

static __device__ __noinline__ bool barrier_wait_long(uint64_t *bar, uint32_t parity, volatile int *broken)
{
    const unsigned long long begin = nanoseconds();
    for (;;) {
        if (barrier_test(bar, parity)) return true;
        if (*broken != 0) return false;
        if (nanoseconds() - begin > kWaitLimit) {
            *broken = 1;
            return false;
        }
    }
}

__device__ __forceinline__ bool barrier_wait(uint64_t *bar, uint32_t parity, volatile int *broken)
{
#pragma unroll 1
    for (int i = 0; i < 16; ++i)
        if (barrier_test(bar, parity)) return true;
    return barrier_wait_long(bar, parity, broken);
}

// After something broke: waits, no longer than the limit either, for what still writes to the block's memory.
static __device__ __noinline__ void barrier_drain(uint64_t *bar, uint32_t parity)
{
    const unsigned long long begin = nanoseconds();
    while (!barrier_test(bar, parity) && nanoseconds() - begin < kWaitLimit) {}
}

__device__ __forceinline__ bool elected()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// ---- copies ------------------------------------------------------------------------------------------

// 128 tokens of a head from `token` on, 64 channels per half, into `dst`; the bytes are counted on `bar`
template <int DP>
__device__ __forceinline__ void load_tile(void *dst, const CUtensorMap *map, int head, int token, int item, uint64_t *bar)
{
#pragma unroll
    for (int half = 0; half < DP / 64; ++half)
        asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                     " [%0], [%1, {%2, %3, %4, %5}], [%6];"
                     ::"r"(shared_address(dst) + half * kHalfBytes), "l"(reinterpret_cast<uint64_t>(map)), "r"(half * 64), "r"(head), "r"(token),
                       "r"(item), "r"(shared_address(bar))
                     : "memory");
}

template <int DP>
constexpr int kTileBytes = DP / 64 * kHalfBytes;

// ---- matrix instructions -------------------------------------------------------------------------------

// Where an operand lies: address, and the distances between its 8-row groups and (rows taken as the sum's axis) its halves.
__device__ __forceinline__ uint64_t operand(uint32_t address, uint32_t half_distance)
{
    return static_cast<uint64_t>((address >> 4) & 0x3fff) | static_cast<uint64_t>((half_distance >> 4) & 0x3fff) << 16 |
           static_cast<uint64_t>(1024 >> 4) << 32 | 1ULL << 46 | 2ULL << 61;
}

// A tile as an operand that is summed over its channels, 16 at a time: channels [16 s, 16 s + 16).  (One thread issues all products, and
// the instructions between them are its time: an operand is one addition.)
__device__ __forceinline__ uint64_t channel_operand(uint32_t tile) { return operand(tile, 16); }
__device__ __forceinline__ uint64_t tile_channels(uint64_t tile, int s) { return tile + static_cast<uint32_t>(((s >> 2) * kHalfBytes + (s & 3) * 32) >> 4); }
// ... over its rows: rows [16 s, 16 s + 16)
__device__ __forceinline__ uint64_t row_operand(uint32_t tile) { return operand(tile, kHalfBytes); }
__device__ __forceinline__ uint64_t tile_rows(uint64_t tile, int s) { return tile + static_cast<uint32_t>(s * 2048 >> 4); }

// Shape and types of a product of 128 rows: float32 sums; b_rows: the second operand is summed over its rows.
template <typename T>
__device__ __forceinline__ uint32_t product_kind(int columns, bool b_rows)
{
    constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
    return 1u << 4 | type << 7 | type << 10 | (b_rows ? 1u << 16 : 0u) | static_cast<uint32_t>(columns >> 3) << 17 | (128u >> 4) << 24;
}

__device__ __forceinline__ void product_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t kind, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(kind), "r"(static_cast<uint32_t>(add))
                 : "memory");
}

// the first operand from tensor memory
__device__ __forceinline__ void product_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t kind, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(kind), "r"(static_cast<uint32_t>(add))
                 : "memory");
}

// `bar` is arrived at when all products issued so far by this thread are done
__device__ __forceinline__ void products_done(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_address(bar)) : "memory");
}

__device__ __forceinline__ void tmem_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// a whole warp: all 512 columns
__device__ __forceinline__ void tmem_take(uint32_t *where)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(shared_address(where)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_give(uint32_t base)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(base) : "memory");
}

#define MA_R8(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), "=r"(x[i + 5]), "=r"(x[i + 6]), "=r"(x[i + 7])
#define MA_W8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])

// 32 columns of the thread's row (a warp: its 32 rows)
__device__ __forceinline__ void tmem_load32(uint32_t at, uint32_t *x)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
                 "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : MA_R8(x, 0), MA_R8(x, 8), MA_R8(x, 16), MA_R8(x, 24)
                 : "r"(at));
}
__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t *x)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : MA_R8(x, 0), MA_R8(x, 8)
                 : "r"(at));
}
__device__ __forceinline__ void tmem_load8(uint32_t at, uint32_t *x)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : MA_R8(x, 0) : "r"(at));
}
__device__ __forceinline__ uint32_t tmem_load1(uint32_t at)
{
    uint32_t x;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(x) : "r"(at));
    return x;
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t *x)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
                 "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::MA_W8(x, 0), MA_W8(x, 8), MA_W8(x, 16), MA_W8(x, 24),
                 "r"(at)
                 : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t *x)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::MA_W8(x, 0),
                 MA_W8(x, 8), "r"(at)
                 : "memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t at, const uint32_t *x)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::MA_W8(x, 0), "r"(at) : "memory");
}
#undef MA_R8
#undef MA_W8

// Waits for the loads before it; the registers pass through it, so that nothing reads them earlier.
#define MA_P8(x, i) "+r"(x[i]), "+r"(x[i + 1]), "+r"(x[i + 2]), "+r"(x[i + 3]), "+r"(x[i + 4]), "+r"(x[i + 5]), "+r"(x[i + 6]), "+r"(x[i + 7])
__device__ __forceinline__ void tmem_loaded32(uint32_t *x)
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" : MA_P8(x, 0), MA_P8(x, 8), MA_P8(x, 16), MA_P8(x, 24)::"memory");
}
__device__ __forceinline__ void tmem_loaded16(uint32_t *x) { asm volatile("tcgen05.wait::ld.sync.aligned;" : MA_P8(x, 0), MA_P8(x, 8)::"memory"); }
__device__ __forceinline__ void tmem_loaded8(uint32_t *x) { asm volatile("tcgen05.wait::ld.sync.aligned;" : MA_P8(x, 0)::"memory"); }
__device__ __forceinline__ void tmem_loaded1(uint32_t &x) { asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(x)::"memory"); }
#undef MA_P8

// ---- arithmetic ---------------------------------------------------------------------------------------

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two float32 at a time.
struct Pair {
    unsigned long long v;
    __device__ __forceinline__ Pair(float low, float high) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(low), "f"(high)); }
    __device__ __forceinline__ void get(float &low, float &high) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(low), "=f"(high) : "l"(v)); }
};
__device__ __forceinline__ Pair pair_fma(Pair a, Pair b, Pair c)
{
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(a.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return a;
}
__device__ __forceinline__ Pair pair_add(Pair a, Pair b)
{
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(a.v) : "l"(a.v), "l"(b.v));
    return a;
}

__device__ __forceinline__ Pair pair_mul(Pair a, Pair b)
{
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(a.v) : "l"(a.v), "l"(b.v));
    return a;
}

__device__ __forceinline__ float reciprocal_fast(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// tanh, in one of two forms by the size of the argument alone: a result does not change with the other scores of a warp, hidden ones among
// them, the backward pass repeats the forward's, and the error stays relative to the score, however far the cap lies above it.
// Up to 0.625: y P(y^2), P of degree 5 with the smallest relative error there, 4e-9 (fitted by reweighted least squares); evaluated in
// float32 it is off by 1.8 * 2^-24, relatively.  Beyond: from one exponential, 1 - 2 / (e^2y + 1), off by a few 2^-24.
constexpr float kSmallTanh = 0.625f;
__device__ constexpr float tanh_term(int i)
{
    return i == 0 ? -5.659989081e-3f : i == 1 ? 2.059098892e-2f : i == 2 ? -5.372106656e-2f : i == 3 ? 1.333112717e-1f : -3.333325982e-1f;
}

// Both forms are there, and no branch per element between them: 2 x 4096 tokens, 16 heads x 128, causal, bfloat16 with a cap of 2 339 us,
// with a branch 543; with a cap of 50, which no score comes near, 229 (scalar polynomials 256).
__device__ __forceinline__ float tanh_form(float y, float small, float large)
{
    float t;
    asm("{\n\t.reg .pred p;\n\t.reg .f32 a;\n\tabs.f32 a, %1;\n\tsetp.le.f32 p, a, %2;\n\tselp.f32 %0, %3, %4, p;\n\t}"
        : "=f"(t)
        : "f"(y), "f"(kSmallTanh), "f"(small), "f"(large));
    return t;
}

__device__ __forceinline__ float tanh_small(float y)
{
    const float u = y * y;
    float r = fmaf(u, tanh_term(0), tanh_term(1));
#pragma unroll
    for (int i = 2; i < 5; ++i) r = fmaf(u, r, tanh_term(i));
    return y * fmaf(u, r, 1.0f);
}
__device__ __forceinline__ Pair tanh_small(Pair y)
{
    const Pair u = pair_mul(y, y);
    Pair r = pair_fma(u, Pair(tanh_term(0), tanh_term(0)), Pair(tanh_term(1), tanh_term(1)));
#pragma unroll
    for (int i = 2; i < 5; ++i) r = pair_fma(u, r, Pair(tanh_term(i), tanh_term(i)));
    return pair_mul(y, pair_fma(u, r, Pair(1.0f, 1.0f)));
}

__device__ __forceinline__ float tanh_one(float y)
{
    return tanh_form(y, tanh_small(y), fmaf(-2.0f, reciprocal_fast(exp2_fast(2.0f * kLog2e * y) + 1.0f), 1.0f));
}

// x[i] = tanh(x[i] * inverse_cap), two at a time.  Scores are mostly well below their cap: where all of a warp's are, the second form and its
// two special-function instructions, which bound the kernels (16 a clock on an SM), are left out.
template <int N>
__device__ __forceinline__ void tanh_all(float *x, float inverse_cap)
{
    float big[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i) big[i % 4] = fmaxf(big[i % 4], fabsf(x[i]));
    const float most = fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3]));
    const Pair by(inverse_cap, inverse_cap);
    if (__all_sync(0xffffffffu, most * inverse_cap <= kSmallTanh)) {
#pragma unroll
        for (int i = 0; i < N; i += 2) tanh_small(pair_mul(Pair(x[i], x[i + 1]), by)).get(x[i], x[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const Pair y = pair_mul(Pair(x[i], x[i + 1]), by);
            float y0, y1, s0, s1, e0, e1;
            y.get(y0, y1);
            tanh_small(y).get(s0, s1);
            pair_mul(y, Pair(2.0f * kLog2e, 2.0f * kLog2e)).get(e0, e1);
            pair_add(Pair(exp2_fast(e0), exp2_fast(e1)), Pair(1.0f, 1.0f)).get(e0, e1);
            pair_fma(Pair(reciprocal_fast(e0), reciprocal_fast(e1)), Pair(-2.0f, -2.0f), Pair(1.0f, 1.0f)).get(e0, e1);
            x[i] = tanh_form(y0, s0, e0);
            x[i + 1] = tanh_form(y1, s1, e1);
        }
    }
}

template <typename T>
__device__ __forceinline__ uint32_t pack_two(float low, float high)
{
    const float x[2] = {low, high};
    return DT<T>::pack(x);
}

template <typename T>
__device__ __forceinline__ void store_eight(T *to, const float *x)
{
    *reinterpret_cast<uint4 *>(to) = make_uint4(pack_two<T>(x[0], x[1]), pack_two<T>(x[2], x[3]), pack_two<T>(x[4], x[5]), pack_two<T>(x[6], x[7]));
}

// zero times every element of a word, added to acc: NaN as soon as one is infinite or NaN
template <typename T>
__device__ __forceinline__ uint32_t taint(uint32_t w, uint32_t acc)
{
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&w), __float2half2_rn(0.0f), *reinterpret_cast<const __half2 *>(&acc));
        return *reinterpret_cast<const uint32_t *>(&r);
    } else {
        const __nv_bfloat162 r =
            __hfma2(*reinterpret_cast<const __nv_bfloat162 *>(&w), __float2bfloat162_rn(0.0f), *reinterpret_cast<const __nv_bfloat162 *>(&acc));
        return *reinterpret_cast<const uint32_t *>(&r);
    }
}

template <typename T>
__device__ __forceinline__ bool tainted(uint32_t acc)
{
    const float a = DT<T>::unpack(acc, 0), b = DT<T>::unpack(acc, 1);
    return a != a || b != b;
}

__device__ __forceinline__ float element(const float4 &x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }
__device__ __forceinline__ int element(const int4 &x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

// Whether a half (of the 16-byte pieces of each 64 channels) of row `row` of a tile holds an infinite or NaN value.
template <typename T, int DP>
__device__ __forceinline__ bool row_tainted(const uint8_t *tile, int row, int part)
{
    uint32_t acc = 0;
#pragma unroll
    for (int half = 0; half < DP / 64; ++half)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int piece = 4 * part + i;
            const uint4 x = *reinterpret_cast<const uint4 *>(tile + half * kHalfBytes + row * 128 + ((piece ^ (row & 7)) << 4));
            acc = taint<T>(x.x, taint<T>(x.y, taint<T>(x.z, taint<T>(x.w, acc))));
        }
    return tainted<T>(acc);
}

// The rows of a tile that a thread's own row sees (or is seen by): those from `from` on, below `to`, and with documents of its id.
struct SeenRows {
    int from, to;
    const int *ids;       // of the tile's rows, or null
    int id;
    __device__ __forceinline__ bool operator()(int j) const { return j >= from && j < to && (ids == nullptr || ids[j] == id); }
};

// The product of the weights in tensor memory (128 x 16 bits per row from `weights` on, RUN of them side by side in every RUN columns) and a
// tile's rows, added to the thread's row of sums at `sums` term by term, leaving out the hidden terms (and no visible one, though its
// weight may be zero): in place of the matrix instruction where the tile holds infinite or NaN values that some rows do not see.  A warp's
// 32 rows; rare, and slow.
template <typename T, int DP, int RUN>
static __device__ __noinline__ void add_rows(uint32_t sums, uint32_t weights, const uint8_t *tile, bool add, SeenRows seen)
{
    for (int c = 0; c < DP; c += 8) {
        uint32_t raw[8] = {};
        if (add) {
            tmem_load8(sums + c, raw);
            tmem_loaded8(raw);
        }
        float acc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = __uint_as_float(raw[i]);
        for (int j = 0; j < kTile; j += 2) {
            uint32_t w = tmem_load1(weights + j / RUN * RUN + j % RUN / 2);
            tmem_loaded1(w);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float x = DT<T>::unpack(w, e);
                const int row = j + e;
                const uint4 y = *reinterpret_cast<const uint4 *>(tile + c / 64 * kHalfBytes + row * 128 + ((c % 64 / 8 ^ (row & 7)) << 4));
                const uint32_t words[4] = {y.x, y.y, y.z, y.w};
                if (seen(row)) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[i] = fmaf(x, DT<T>::unpack(words[i / 2], i % 2), acc[i]);
                }
            }
            __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = __float_as_uint(acc[i]);
        tmem_store8(sums + c, raw);
    }
    tmem_stored();
}

// ---- masks by tiles ------------------------------------------------------------------------------------

// Keys that query n sees are those below this (and, with documents, of its id).
__device__ __forceinline__ int key_limit(const GlobalMask &m, int n)
{
    return m.causal ? min(m.len, max(max(n + m.shift + 1, m.prefix), 0)) : m.len;
}

enum TileState { kHidden, kPartial, kWhole };

// By the tokens' distance: none, in a sequence, on a map.
enum GlobalBias { kNoBias, kSequenceBias, kMapBias };

// What the queries [n0, n0 + 128) see of the keys [j0, j0 + 128).
__device__ __forceinline__ int tile_state(const GlobalMask &m, int N, int n0, int j0, const DocRange *qr, const DocRange *kr)
{
    if (n0 >= N || j0 >= key_limit(m, min(n0 + kTile, N) - 1)) return kHidden;
    const bool whole = j0 + kTile <= key_limit(m, n0);
    if (kr == nullptr) return whole ? kWhole : kPartial;
    const DocRange q = *qr, k = *kr;
    if (k.high < q.low || k.low > q.high || q.high < 0 || k.high < 0) return kHidden;
    return whole && q.pure && k.pure && q.low == q.high && k.low == k.high ? kWhole : kPartial;
}

// Whether queries whose last key tile is before `end` see anything of key tile t; with documents by their ranges.
__device__ __forceinline__ bool tile_seen(int t, int end, const DocRange *qr, const DocRange *kr)
{
    if (t >= end) return false;
    if (kr == nullptr) return true;
    const DocRange q = *qr, k = kr[t];
    return !(k.high < q.low || k.low > q.high || q.high < 0 || k.high < 0);
}

// ---- host ----------------------------------------------------------------------------------------------

// Whether the matrix kernels take a tensor: 16-byte aligned rows, no dimension repeated by a stride of zero.
inline bool rows_fit(const void *base, const long long (&stride)[3], int B, int rows, int heads)
{
    const int sizes[3] = {B, rows, heads};
    if (reinterpret_cast<uintptr_t>(base) % 16 != 0) return false;
    for (int i = 0; i < 3; ++i)
        if (sizes[i] > 1 && (stride[i] <= 0 || stride[i] % 8 != 0 || stride[i] >= (1LL << 38))) return false;
    return true;
}

// Builds by what a score goes through: calls f(channels of a tile, capped, bias) as types.
template <typename F>
cudaError_t by_scores(const GlobalParams &p, F f)
{
    const auto bias = [&](auto width, auto cap) {
        if (p.slopes == nullptr) return f(width, cap, std::integral_constant<GlobalBias, kNoBias>());
        if (p.width == 1) return f(width, cap, std::integral_constant<GlobalBias, kSequenceBias>());
        return f(width, cap, std::integral_constant<GlobalBias, kMapBias>());
    };
    const auto cap = [&](auto width) { return p.cap != 0.0f ? bias(width, std::true_type()) : bias(width, std::false_type()); };
    return p.d <= 64 ? cap(std::integral_constant<int, 64>()) : cap(std::integral_constant<int, 128>());
}

template <typename T>
cudaError_t run_global_forward(const GlobalParams &p, const GlobalMaps &maps, cudaStream_t stream);
cudaError_t run_global_token(const GlobalParams &p, int dtype, cudaStream_t stream);
template <typename T>
cudaError_t run_global_backward(const GlobalParams &p, const GlobalMaps &maps, cudaStream_t stream);


}  // namespace matchattn
