// Norm of every head of q and k and its rotation by the token's position, one pass over both (matchattn_norm_rotary_*).
//
//   u = x * rsqrt(mean(x^2) + eps),  g = u * weight
//   y[i]         = g[i] cos(a_i) - g[i + rot/2] sin(a_i)        i < rot/2
//   y[i + rot/2] = g[i + rot/2] cos(a_i) + g[i] sin(a_i)        channels from rot on: y = g
//
// The angle a_i is position * frequency.  A frequency is a 64-bit fraction of a turn per position: the product with the
// position wraps at whole turns by itself, so what is left is exact but for the table's rounding, 2^-65 turns per position, however far
// that lies (a float32 product is off by 0.06 rad at position 10^6).  Its upper half goes to sincospif as a float32 of half turns: 2^-26
// turns.
//
// Backward, from dy and x: dg = dy rotated back, dw = sum dg * u, e = dg * weight, dx = r (e - u mean(e u)).
//
// Bound by memory: x in, y out (backward: x, dy in, dx out).  A group of lanes owns a token's row of a head: a lane holds V
// channels and the V they are paired with, so the rotation stays in the lane, a row is read once, and mean and rotation work from
// registers; V channels are one load of up to 16 bytes, and the next row is on its way while one is computed.  The groups of a warp take
// heads of the same token side by side and in turn: a head's rows are one run of memory, and the token's angles (a sincospif per pair,
// as many instructions as a head's row altogether) are formed once, each group a share.  All sums are float32, results are
// rounded once.  Measured, one B200: 16384 tokens, 40 heads x 128, bfloat16 69 us (4.9 TB/s), backward 106 us (4.7 TB/s) and 6 for the
// weights; 384 x 384 tokens, 16 heads x 16, float16 55 us (2.7 TB/s; 511 instructions per warp and row, issue 68 %).
// The weights' gradients are summed per lane over the rows of a block (float32, a dozen of them or so), then over the block, then over the
// blocks by a second kernel (both in float64, whose few additions cost nothing), always in the same order: no atomics.
#include "matchattn_kernels.cuh"

#include <type_traits>

namespace matchattn {
namespace {

constexpr int kNormThreads = 128;
constexpr int kNormHeads = 8;            // heads that a group takes in turn at most

struct NormSide {            // queries or keys
    const void *x, *w, *dy;
    void *y, *dw;            // forward: the result; backward: dx
    float *partial;          // [blocks, d]
    long long stride[3];
    int heads, chunks, per;  // heads of a token: `chunks` groups of `per`
    int blocks;
};

struct NormParams {
    NormSide side[2];
    const void *positions;
    const unsigned long long *freqs;
    long long pos_item;      // positions per item (0: all items share them)
    int pos64, axes, rot, B, N, d, w32;
    float eps, inv_d;
};

// V channels as they lie in memory
template <typename T, int V>
struct Run {
    static constexpr int kWords = V == 1 ? 1 : V * static_cast<int>(sizeof(T)) / 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void load(const T *p, bool there)
    {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
        if (!there) return;
        if constexpr (V == 1) {
            w[0] = __float_as_uint(load_one<T>(p));
        } else if constexpr (kWords == 4) {
            const uint4 t = *reinterpret_cast<const uint4 *>(p);
            w[0] = t.x, w[1] = t.y, w[2] = t.z, w[3] = t.w;
        } else {
            const uint2 t = *reinterpret_cast<const uint2 *>(p);
            w[0] = t.x, w[1] = t.y;
        }
    }
    __device__ __forceinline__ float get(int i) const
    {
        if constexpr (V == 1) return __uint_as_float(w[0]);
        else return DT<T>::unpack(w[i / DT<T>::kElemsPerWord], i % DT<T>::kElemsPerWord);
    }
};

template <typename T, int V>
__device__ __forceinline__ void store_run(T *p, const float (&x)[V])
{
    constexpr int bytes = V * sizeof(T);
    if constexpr (V == 1) {
        store_one<T>(p, x[0]);
    } else {
        uint32_t w[bytes / 4];
#pragma unroll
        for (int i = 0; i < bytes / 4; ++i) w[i] = DT<T>::pack(x + i * DT<T>::kElemsPerWord);
        if constexpr (bytes == 16) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
    }
}

// V channels of a weight in T or float32
template <typename T, int V>
__device__ __forceinline__ void load_weight(const NormParams &p, const void *w, int c, float (&x)[V])
{
    if (w == nullptr) {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = 1.0f;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = p.w32 ? static_cast<const float *>(w)[c + i] : load_one<T>(static_cast<const T *>(w) + c + i);
    }
}

template <int S, int V>
struct Turns {
    float cosine[S][V], sine[S][V];
};

// A group's token and first head.
struct Place {
    unsigned token;
    int b, n, h0;
    bool on;
};

// first channel of a slot's two runs; slots below `paired` are rotated
struct Slot {
    int a, b;
};
template <int V>
__device__ __forceinline__ Slot slot_of(int s, int paired, int rot)
{
    return s < paired ? Slot{s * V, s * V + rot / 2} : Slot{rot + 2 * (s - paired) * V, rot + (2 * (s - paired) + 1) * V};
}

__device__ __forceinline__ void turn_of(const NormParams &p, const long long (&pos)[2], int pair, float &cosine, float &sine)
{
    const int per_axis = p.rot / 2 / p.axes;
    const unsigned long long turn = p.freqs[pair] * static_cast<unsigned long long>(pair >= per_axis ? pos[1] : pos[0]);
    sincospif(static_cast<float>(static_cast<int>(turn >> 32)) * 4.656612873077393e-10f, &sine, &cosine);
}

// Of the V pairs of a lane's slot each of V / SHARE groups of lanes, which have the same token, forms SHARE.
template <int V, int SHARE>
__device__ __forceinline__ void share_turns(const NormParams &p, const long long (&pos)[2], int slot, bool turned, int member, int lanes, Turns<1, V> &t)
{
    float cosine[SHARE], sine[SHARE];
#pragma unroll
    for (int m = 0; m < SHARE; ++m) {
        cosine[m] = 1.0f;
        sine[m] = 0.0f;
        if (turned) turn_of(p, pos, slot * V + member * SHARE + m, cosine[m], sine[m]);
    }
    const int base = (threadIdx.x & 31) - member * lanes;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        t.cosine[0][i] = __shfl_sync(0xffffffffu, cosine[i % SHARE], base + i / SHARE * lanes);
        t.sine[0][i] = __shfl_sync(0xffffffffu, sine[i % SHARE], base + i / SHARE * lanes);
    }
}

// lane: of its group; member: the group's place among the `spread` groups that take the heads of a token together
template <int V, int S>
__device__ __forceinline__ void find_turns(const NormParams &p, const long long (&pos)[2], int lane, int lanes, int member, int spread, int paired,
                                           Turns<S, V> &t)
{
    if (p.rot == 0) return;
    if constexpr (S == 1 && V > 1) {
        const bool turned = lane < paired;
        if (spread >= V) share_turns<V, 1>(p, pos, lane, turned, member, lanes, t);
        else if (spread * 2 == V) share_turns<V, 2>(p, pos, lane, turned, member, lanes, t);
        else if (spread * 4 == V) share_turns<V, 4>(p, pos, lane, turned, member, lanes, t);
        else share_turns<V, V>(p, pos, lane, turned, member, lanes, t);
    } else {
#pragma unroll
        for (int k = 0; k < S; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                t.cosine[k][i] = 1.0f;
                t.sine[k][i] = 0.0f;
                if (lane + k * lanes < paired) turn_of(p, pos, (lane + k * lanes) * V + i, t.cosine[k][i], t.sine[k][i]);
            }
    }
}

__device__ __forceinline__ float group_sum(float v, int lanes)
{
    for (int o = lanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// T: element, V: channels per run, S: slots per lane, BACK: the backward pass
template <typename T, int V, int S, bool BACK>
__global__ void __launch_bounds__(kNormThreads, BACK || S > 1 ? 4 : 6) norm_rotary_kernel(const NormParams p, int lanes, int spread)
{
    chain_begin();
    __shared__ float reduced[BACK ? kNormThreads * 2 * V : 1];
    const int second = blockIdx.x >= p.side[0].blocks;
    const NormSide &s = p.side[second];
    const int block = blockIdx.x - (second ? p.side[0].blocks : 0);
    const int lane = threadIdx.x & (lanes - 1), member = threadIdx.x / lanes & (spread - 1);
    const int group = threadIdx.x / (lanes * spread), groups = kNormThreads / (lanes * spread);
    const int paired = p.rot / (2 * V);
    const unsigned items = static_cast<unsigned>(p.B) * p.N * s.chunks;
    float wa[S][V], wb[S][V], dwa[S][V], dwb[S][V];
    bool has_a[S], has_b[S];
    Slot at[S];
#pragma unroll
    for (int k = 0; k < S; ++k) {
        at[k] = slot_of<V>(lane + k * lanes, paired, p.rot);
        has_a[k] = at[k].a + V <= p.d;
        has_b[k] = at[k].b + V <= p.d;
#pragma unroll
        for (int i = 0; i < V; ++i) wa[k][i] = wb[k][i] = dwa[k][i] = dwb[k][i] = 0.0f;
        if (has_a[k]) load_weight<T, V>(p, s.w, at[k].a, wa[k]);
        if (has_b[k]) load_weight<T, V>(p, s.w, at[k].b, wb[k]);
    }
    // the next row, and the next token's position, are on their way while a row is computed
    Run<T, V> next_x[S][2], next_g[S][2];
    long long next_pos[2] = {0, 0};
    const auto place_of = [&](unsigned item) {
        Place at;
        at.on = item < items;
        at.token = at.on ? item / s.chunks : 0;
        at.h0 = (at.on ? static_cast<int>(item - at.token * s.chunks) * s.per * spread : 0) + member;
        at.b = static_cast<int>(at.token / p.N);
        at.n = static_cast<int>(at.token) - at.b * p.N;
        return at;
    };
    const auto fetch = [&](const Place &to, int i0) {
        const int head = to.h0 + i0 * spread;
        const bool there = to.on && head < s.heads;
        const T *x = static_cast<const T *>(s.x) + to.b * s.stride[0] + to.n * s.stride[1] + head * s.stride[2];
        const T *dy = static_cast<const T *>(s.dy) + (static_cast<long long>(to.token) * s.heads + head) * p.d;
#pragma unroll
        for (int k = 0; k < S; ++k) {
            next_x[k][0].load(x + at[k].a, there && has_a[k]);
            next_x[k][1].load(x + at[k].b, there && has_b[k]);
            if constexpr (BACK) {
                next_g[k][0].load(dy + at[k].a, there && has_a[k]);
                next_g[k][1].load(dy + at[k].b, there && has_b[k]);
            }
        }
        if (i0 == 0 && p.rot > 0) {
#pragma unroll
            for (int a = 0; a < 2; ++a)
                if (a < p.axes) {
                    const long long i = to.b * p.pos_item + static_cast<long long>(to.n) * p.axes + a;
                    next_pos[a] = p.pos64 ? static_cast<const long long *>(p.positions)[i] : static_cast<const int *>(p.positions)[i];
                }
        }
    };
    // every group of a warp makes the same number of rounds (their sums are taken by the whole warp)
    const unsigned step = static_cast<unsigned>(s.blocks) * groups;
    Place next = place_of(static_cast<unsigned>(block) * groups + group);
    fetch(next, 0);
    for (unsigned first = static_cast<unsigned>(block) * groups; first < items; first += step) {
        const Place now = next;
        const long long flat = static_cast<long long>(now.token) * s.heads * p.d;
        Turns<S, V> t;
        find_turns<V, S>(p, next_pos, lane, lanes, member, spread, paired, t);
        next = place_of(first + step + group);
#pragma unroll 1
        for (int i0 = 0; i0 < s.per; ++i0) {
            const int head = now.h0 + i0 * spread;
            const bool live = now.on && head < s.heads;
            float xa[S][V], xb[S][V], ga[S][V], gb[S][V], square = 0.0f;
#pragma unroll
            for (int k = 0; k < S; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    xa[k][i] = next_x[k][0].get(i), xb[k][i] = next_x[k][1].get(i);
                    if constexpr (BACK) ga[k][i] = next_g[k][0].get(i), gb[k][i] = next_g[k][1].get(i);
                }
            if (i0 + 1 < s.per) fetch(now, i0 + 1);
            else fetch(next, 0);
#pragma unroll
            for (int k = 0; k < S; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) square = fmaf(xa[k][i], xa[k][i], fmaf(xb[k][i], xb[k][i], square));
            const float r = rsqrtf(fmaf(group_sum(square, lanes), p.inv_d, p.eps));
            T *out = static_cast<T *>(s.y) + flat + static_cast<long long>(head) * p.d;
            if constexpr (!BACK) {
#pragma unroll
                for (int k = 0; k < S; ++k) {
                    float ya[V], yb[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float u = xa[k][i] * r * wa[k][i], v = xb[k][i] * r * wb[k][i];
                        ya[i] = lane + k * lanes < paired ? u * t.cosine[k][i] - v * t.sine[k][i] : u;
                        yb[i] = lane + k * lanes < paired ? v * t.cosine[k][i] + u * t.sine[k][i] : v;
                    }
                    if (live && has_a[k]) store_run<T, V>(out + at[k].a, ya);
                    if (live && has_b[k]) store_run<T, V>(out + at[k].b, yb);
                }
            } else {
                float dot = 0.0f;
#pragma unroll
                for (int k = 0; k < S; ++k)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const bool turned = lane + k * lanes < paired;
                        const float da = turned ? ga[k][i] * t.cosine[k][i] + gb[k][i] * t.sine[k][i] : ga[k][i];
                        const float db = turned ? gb[k][i] * t.cosine[k][i] - ga[k][i] * t.sine[k][i] : gb[k][i];
                        xa[k][i] *= r, xb[k][i] *= r;
                        if (live) {
                            dwa[k][i] = fmaf(da, xa[k][i], dwa[k][i]);
                            dwb[k][i] = fmaf(db, xb[k][i], dwb[k][i]);
                        }
                        ga[k][i] = da * wa[k][i], gb[k][i] = db * wb[k][i];
                        dot = fmaf(ga[k][i], xa[k][i], fmaf(gb[k][i], xb[k][i], dot));
                    }
                const float mean = group_sum(dot, lanes) * p.inv_d;
#pragma unroll
                for (int k = 0; k < S; ++k) {
                    float da[V], db[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        da[i] = r * (ga[k][i] - xa[k][i] * mean);
                        db[i] = r * (gb[k][i] - xb[k][i] * mean);
                    }
                    if (live && has_a[k]) store_run<T, V>(out + at[k].a, da);
                    if (live && has_b[k]) store_run<T, V>(out + at[k].b, db);
                }
            }
        }
    }
    if constexpr (BACK) {
        if (s.partial == nullptr) return;
#pragma unroll
        for (int k = 0; k < S; ++k) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < V; ++i) {
                reduced[i * kNormThreads + threadIdx.x] = dwa[k][i];
                reduced[(V + i) * kNormThreads + threadIdx.x] = dwb[k][i];
            }
            __syncthreads();
            // thread (run element, lane): the sum over the groups
            for (int e = threadIdx.x; e < 2 * V * lanes; e += kNormThreads) {
                const int l = e & (lanes - 1), i = e / lanes;
                const Slot c = slot_of<V>(l + k * lanes, paired, p.rot);
                const int channel = i < V ? c.a + i : c.b + i - V;
                double sum = 0.0;
                for (int g = 0; g < kNormThreads / lanes; ++g) sum += reduced[i * kNormThreads + g * lanes + l];
                if (channel < p.d) s.partial[static_cast<long long>(block) * p.d + channel] = static_cast<float>(sum);
            }
        }
    }
}

// dw[c] = sum over the blocks of partial[block][c], in a fixed order; 32 channels x 32 rows of threads
template <typename T>
__global__ void __launch_bounds__(1024) norm_weight_kernel(const NormParams p)
{
    chain_begin();
    __shared__ double sums[32][33];
    const NormSide &s = p.side[blockIdx.y];
    if (s.partial == nullptr) return;
    const int c = blockIdx.x * 32 + threadIdx.x;
    double sum = 0.0;
    if (c < p.d)
        for (int i = threadIdx.y; i < s.blocks; i += 32) sum += s.partial[static_cast<long long>(i) * p.d + c];
    sums[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    sum = sums[threadIdx.x][threadIdx.y];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int out = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && out < p.d) {
        if (p.w32) static_cast<float *>(s.dw)[out] = static_cast<float>(sum);
        else store_one<T>(static_cast<T *>(s.dw) + out, static_cast<float>(sum));
    }
}

// The blocks of one side, and how its heads are cut: `spread` at a time, `per` times in turn.  Heads in turn share the angles; a
// small call spreads them instead, so that the chip fills.  No more than `most` blocks, each of which takes items in turn.
void lay_out(NormSide &s, long long tokens, int groups, int spread, long long wanted, long long most)
{
    const int turns = (s.heads + spread - 1) / spread;
    s.per = turns < kNormHeads ? turns : kNormHeads;
    while (s.per > 1 && tokens * ((turns + s.per - 1) / s.per) < wanted * groups) s.per = (s.per + 1) / 2;
    s.chunks = (turns + s.per - 1) / s.per;
    const long long items = tokens * s.chunks, blocks = (items + groups - 1) / groups;
    s.blocks = static_cast<int>(blocks < most ? blocks : most);
}

constexpr int kNormBackBlocks = 4, kNormForwardBlocks = 6;       // blocks per SM and side at most

template <typename T, int V, int S>
cudaError_t run_norm_slots(NormParams &p, bool back, cudaStream_t stream)
{
    const int slots = ((p.d + V - 1) / V + 1) / 2;
    int lanes = 1;
    while (lanes < 32 && lanes * S < slots) lanes *= 2;
    // as many heads side by side as share a warp, up to one per pair of a lane: they read and write one run of memory, and each
    // forms its share of the token's angles
    int spread = 1;
    while (S == 1 && V > 1 && spread < V && spread * lanes < 32 && spread < p.side[0].heads) spread *= 2;
    const int groups = kNormThreads / (lanes * spread);
    int blocks = 0;
    for (NormSide &s : p.side) {
        if (s.heads > 0) lay_out(s, static_cast<long long>(p.B) * p.N, groups, spread, 1LL * sm_count() * kNormBackBlocks,
                                  1LL * sm_count() * (back ? kNormBackBlocks : kNormForwardBlocks));
        blocks += s.blocks;
    }
    const cudaError_t err = back ? launch_chained(norm_rotary_kernel<T, V, S, true>, dim3(blocks), kNormThreads, 0, stream, p, lanes, spread)
                                 : launch_chained(norm_rotary_kernel<T, V, S, false>, dim3(blocks), kNormThreads, 0, stream, p, lanes, spread);
    if (err != cudaSuccess || (p.side[0].partial == nullptr && p.side[1].partial == nullptr)) return err;
    return launch_chained(norm_weight_kernel<T>, dim3((p.d + 31) / 32, 2), dim3(32, 32), 0, stream, p);
}

bool fits(const NormParams &p, int V, size_t size, bool back)
{
    if (p.d % V != 0 || p.rot % (2 * V) != 0) return false;
    for (const NormSide &s : p.side) {
        if (s.heads == 0) continue;
        for (const void *a : {s.x, static_cast<const void *>(s.y), back ? s.dy : s.x})
            if (reinterpret_cast<uintptr_t>(a) % (V * size) != 0) return false;
        for (long long t : s.stride)
            if (t % V != 0) return false;
    }
    return true;
}

// The widest runs that the sizes and addresses allow: 16 bytes, 8, single elements.
template <typename T>
cudaError_t run_norm(NormParams &p, bool back, cudaStream_t stream)
{
    constexpr int wide = 16 / sizeof(T);
    if (fits(p, wide, sizeof(T), back) && p.d <= 64 * wide) return run_norm_slots<T, wide, 1>(p, back, stream);
    if constexpr (sizeof(T) == 2) {
        if (fits(p, 4, sizeof(T), back)) return run_norm_slots<T, 4, 1>(p, back, stream);
    }
    return p.d <= 64 ? run_norm_slots<T, 1, 1>(p, back, stream) : run_norm_slots<T, 1, 4>(p, back, stream);
}

int check_norm(const matchattn_norm_args *a)
{
    if (a == nullptr || !a->q || (a->hk > 0 && !a->k)) return MATCHATTN_ERR_NULL;
    if (a->rot > 0 && (!a->positions || !a->freqs)) return MATCHATTN_ERR_NULL;
    if (a->B <= 0 || a->N <= 0 || a->h <= 0 || a->hk < 0 || a->d <= 0 || a->d > MATCHATTN_MAX_DENSE_D || a->rot < 0 || a->rot > a->d ||
        a->axes < 1 || a->axes > 2 || a->rot % (2 * a->axes) != 0 || !(a->eps >= 0.0f) || a->eps > 3.402823466e38f)
        return MATCHATTN_ERR_SHAPE;
    if (a->dtype < MATCHATTN_F32 || a->dtype > MATCHATTN_BF16) return MATCHATTN_ERR_DTYPE;
    if (a->weight_dtype != MATCHATTN_F32 && a->weight_dtype != a->dtype) return MATCHATTN_ERR_DTYPE;
    const uintptr_t size = a->dtype == MATCHATTN_F32 ? 4 : 2, wsize = a->weight_dtype == MATCHATTN_F32 ? 4 : 2;
    for (const void *t : {a->q, a->k})
        if (reinterpret_cast<uintptr_t>(t) % size != 0) return MATCHATTN_ERR_ALIGN;
    for (const void *t : {a->q_weight, a->k_weight})
        if (reinterpret_cast<uintptr_t>(t) % wsize != 0) return MATCHATTN_ERR_ALIGN;
    if (reinterpret_cast<uintptr_t>(a->freqs) % 8 != 0 || reinterpret_cast<uintptr_t>(a->positions) % (a->positions_64 ? 8 : 4) != 0)
        return MATCHATTN_ERR_ALIGN;
    if (a->h > (1 << 20) || a->hk > (1 << 20) || 1LL * a->B * a->N * ((a->h > a->hk ? a->h : a->hk)) > (1LL << 31) - 1)
        return MATCHATTN_ERR_TOO_LARGE;
    return MATCHATTN_OK;
}

NormParams norm_params(const matchattn_norm_args *a)
{
    NormParams p{};
    const void *x[2] = {a->q, a->k}, *w[2] = {a->q_weight, a->k_weight};
    const long long *stride[2] = {a->q_stride, a->k_stride};
    const int heads[2] = {a->h, a->hk};
    for (int i = 0; i < 2; ++i) {
        p.side[i].x = x[i];
        p.side[i].w = w[i];
        p.side[i].heads = heads[i];
        for (int j = 0; j < 3; ++j) p.side[i].stride[j] = stride[i][j];
    }
    p.positions = a->positions;
    p.freqs = static_cast<const unsigned long long *>(a->freqs);
    p.pos_item = a->positions_per_item;
    p.pos64 = a->positions_64;
    p.axes = a->axes;
    p.rot = a->rot;
    p.B = a->B, p.N = a->N, p.d = a->d;
    p.w32 = a->weight_dtype == MATCHATTN_F32;
    p.eps = a->eps;
    p.inv_d = 1.0f / static_cast<float>(a->d);
    return p;
}

cudaError_t run_norm_type(NormParams &p, int dtype, bool back, cudaStream_t stream)
{
    switch (dtype) {
    case MATCHATTN_F32: return run_norm<float>(p, back, stream);
    case MATCHATTN_F16: return run_norm<__half>(p, back, stream);
    default: return run_norm<__nv_bfloat16>(p, back, stream);
    }
}

}  // namespace
}  // namespace matchattn

extern "C" int matchattn_norm_rotary_forward(const matchattn_norm_args *a, void *q_out, void *k_out, void *cuda_stream)
{
    using namespace matchattn;
    const int bad = check_norm(a);
    if (bad != MATCHATTN_OK) return bad;
    if (!q_out || (a->hk > 0 && !k_out)) return MATCHATTN_ERR_NULL;
    NormParams p = norm_params(a);
    p.side[0].y = q_out;
    p.side[1].y = k_out;
    return status_of(run_norm_type(p, a->dtype, false, static_cast<cudaStream_t>(cuda_stream)));
}

extern "C" size_t matchattn_norm_rotary_scratch_bytes(int d)
{
    if (d <= 0 || d > MATCHATTN_MAX_DENSE_D) return 0;
    return 2 * sizeof(float) * static_cast<size_t>(d) * matchattn::sm_count() * matchattn::kNormBackBlocks;
}

extern "C" int matchattn_norm_rotary_backward(const matchattn_norm_args *a, const void *d_q_out, const void *d_k_out, void *d_q, void *d_k,
                                              void *d_q_weight, void *d_k_weight, void *scratch, size_t scratch_bytes, void *cuda_stream)
{
    using namespace matchattn;
    const int bad = check_norm(a);
    if (bad != MATCHATTN_OK) return bad;
    if (!d_q_out || !d_q || (a->hk > 0 && (!d_k_out || !d_k))) return MATCHATTN_ERR_NULL;
    if ((d_q_weight && !a->q_weight) || (d_k_weight && !a->k_weight)) return MATCHATTN_ERR_NULL;
    if (d_q_weight || d_k_weight) {
        if (!scratch) return MATCHATTN_ERR_NULL;
        if (scratch_bytes < matchattn_norm_rotary_scratch_bytes(a->d)) return MATCHATTN_ERR_SCRATCH_LIMIT;
        if (reinterpret_cast<uintptr_t>(scratch) % 4 != 0) return MATCHATTN_ERR_ALIGN;
    }
    NormParams p = norm_params(a);
    p.side[0].dy = d_q_out, p.side[1].dy = d_k_out;
    p.side[0].y = d_q, p.side[1].y = d_k;
    p.side[0].dw = d_q_weight, p.side[1].dw = a->hk > 0 ? d_k_weight : nullptr;
    float *room = static_cast<float *>(scratch);
    for (NormSide &s : p.side) {
        if (s.dw != nullptr) s.partial = room;
        if (room != nullptr) room += static_cast<size_t>(a->d) * sm_count() * kNormBackBlocks;
    }
    return status_of(run_norm_type(p, a->dtype, true, static_cast<cudaStream_t>(cuda_stream)));
}
