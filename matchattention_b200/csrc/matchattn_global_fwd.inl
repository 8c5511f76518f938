// Dense attention, forward, 16-bit types of up to 128 channels, on the matrix units.  Included once per type with MATCHATTN_T
// defined.
//
// A block owns 256 queries of a head as two tiles of 128 (or one tile, when the call has too few for the chip).  Warps 0-7 and 8-15
// take the softmax of one tile each, a thread 64 of the 128 scores of a query; warp 16 copies tiles of K and V into a ring of
// buffers (tensor memory accelerator); one thread of warp 17 issues the products: S = Q K^T into tensor memory, and O += P V with P from
// tensor memory, where it overwrites the scores.  While one tile's threads take exponentials the matrix unit works on the other's.
//
// The softmax keeps a reference per row, not the running maximum itself: probabilities are taken with the reference as it stands,
// and O, the sum and the probabilities only change to a new one when a score exceeds it by 2^8.  They stay below 2^8, O in
// tensor memory is hardly ever touched between products, and nothing waits for a maximum.  float16 has few exponents: P, the sum and O are
// held times 2^7 there, the room that the type leaves above 2^8, and over keys without end, whose small weights add up, times 2^11,
// with a reference that moves at 2^4 (for every call that would cost: 48 x 48 tokens with a map bias 62 us for 51).
// P is rounded to the type of V (a half step of it, relative, as torch rounds a softmax's result; the matrix unit takes both operands in one
// type, and a second term of P would be a product more); scores, reference, sums and O are float32.  For training O is divided by the sum of the rounded probabilities: their errors then weigh differences of values and not
// the values (8160 tokens of 8 heads x 16, float16: 2.8e-4 from the exact result, 2.9e-4 without), which the row sums of the backward
// pass build on.  Elsewhere by the sum itself: the second sum costs 5 to 10 %.
//
// Measured, one B200: 8192 tokens, 32 heads x 128 on 8 key heads, bfloat16, causal 617 us a call (0.89 PFLOP/s, 0.54 of the measured rate of a
// library product).  Calls of one input in a row took 566, and 467 with the softmax taken out: scores read both of their operands from
// shared memory at its full rate, beside the copies into it.  48 x 48 tokens x 2, 4 heads x 32, float16, map bias 51 us: one tile per
// block and SM, eighteen dependent steps of 2.8 us.
//
// A probability that the mask makes zero meets V all the same in the product, and 0 * NaN is NaN: where a tile is partly
// hidden, its V is looked through first, and one with infinite or NaN values is added term by term.
#include "matchattn_global_mma.cuh"

namespace matchattn {
namespace {

constexpr int kForwardThreads = 576;

template <int DP>
struct ForwardShared {
    static constexpr int kStages = DP == 128 ? 4 : 6;
    uint8_t q[2][kTileBytes<DP>];
    uint8_t kv[kStages][kTileBytes<DP>];
    float4 across[16][16], down[16][16];           // per softmax warp, its 64 keys: columns and rows on the map
    int4 docs[16][16];
    float high[2][2][2][kTile], weight[2][2][kTile];      // by turns: tile, half, row
    uint64_t agreed[2][4], q_full, kv_full[kStages], kv_empty[kStages], s_full[2], p_full[2], o_full[2];
    uint32_t tmem;
    uint64_t looked[2];                  // a warpgroup has looked through a tile of V
    int broken, by_hand[2], odd[2][3];
};

template <typename T, int DP, bool CAP, GlobalBias BIAS>
__global__ void __launch_bounds__(kForwardThreads, 1) global_forward_kernel(const GlobalParams p, const __grid_constant__ GlobalMaps maps)
{
    chain_begin();
    constexpr int STAGES = ForwardShared<DP>::kStages;
    constexpr bool GENERAL = CAP || BIAS != kNoBias;
    // log2 of what P is held by, and of what it may exceed that by: together at most 2^15 in float16
    const float held = std::is_same<T, __half>::value ? p.held : 0.0f, slack = std::is_same<T, __half>::value ? 15.0f - held : 8.0f;
    extern __shared__ uint8_t raw_shared[];
    ForwardShared<DP> &sh = *reinterpret_cast<ForwardShared<DP> *>(raw_shared + (1024 - (shared_address(raw_shared) & 1023)) % 1024);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int lot = p.B * p.h * p.splits, turn = blockIdx.x / lot, bh = blockIdx.x % lot % (p.B * p.h), split = blockIdx.x % lot / (p.B * p.h);
    const int b = bh / p.h, head = bh - b * p.h, kh = head / p.g;
    // the last queries of a causal call see most: their blocks begin first
    const int n0 = (gridDim.x / lot - 1 - turn) * p.block_rows;
    const GlobalMask mask = global_mask(p, b);
    const int key_tiles = (p.M + kTile - 1) / kTile, query_tiles = (p.N + kTile - 1) / kTile;
    const DocRange *kr = p.q_docs ? p.ranges + p.B * query_tiles + b * key_tiles : nullptr;
    const DocRange *qr = p.q_docs ? p.ranges + b * query_tiles + n0 / kTile : nullptr;
    const int tiles = p.block_rows / kTile;          // 1 or 2
    const auto state = [&](int w, int t) {
        if (w >= tiles) return static_cast<int>(kHidden);
        return tile_state(mask, p.N, n0 + w * kTile, t * kTile, qr ? qr + w : nullptr, kr ? kr + t : nullptr);
    };
    const int end = (key_limit(mask, min(n0 + p.block_rows, p.N) - 1) + kTile - 1) / kTile;
    // the same in short, for the two threads that copy and multiply: key tiles that a query tile sees any of
    const int ends[2] = {(key_limit(mask, min(n0 + kTile, p.N) - 1) + kTile - 1) / kTile, tiles > 1 && n0 + kTile < p.N ? end : 0};
    const auto seen = [&](int w, int t) { return tile_seen(t, ends[w], qr ? qr + w : nullptr, kr); };
    const int t_begin = split * p.tiles_per_split, t_end = p.splits > 1 ? min(end, t_begin + p.tiles_per_split) : end;

    if (tid == 0) {
        barrier_init(&sh.q_full, 1);
        for (int i = 0; i < STAGES; ++i) {
            barrier_init(&sh.kv_full[i], 1);
            barrier_init(&sh.kv_empty[i], 1);
        }
        for (int w = 0; w < 2; ++w) {
            barrier_init(&sh.s_full[w], 1);
            barrier_init(&sh.p_full[w], 8);
            for (int i = 0; i < 4; ++i) barrier_init(&sh.agreed[w][i], 2);
            barrier_init(&sh.o_full[w], 1);
            barrier_init(&sh.looked[w], 8);
            for (int i = 0; i < 3; ++i) sh.odd[w][i] = 0;
        }
        sh.broken = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 17) tmem_take(&sh.tmem);
    tmem_before();
    __syncthreads();
    tmem_after();
    const uint32_t tmem = sh.tmem;

    if (warp == 16) {
        // ---- copies: Q, then K and V of every tile that one of the two query tiles sees
        if (elected()) {
            barrier_expect(&sh.q_full, tiles * kTileBytes<DP>);
            for (int w = 0; w < tiles; ++w) load_tile<DP>(sh.q[w], &maps.q, head, n0 + w * kTile, b, &sh.q_full);
            int n = 0;           // tiles copied, K and V counted apart
            bool good = true;
            for (int t = t_begin; t < t_end && good; ++t) {
                if (!seen(0, t) && !seen(1, t)) continue;
                for (int i = 0; i < 2 && good; ++i, ++n) {
                    const int s = n % STAGES;
                    if (n >= STAGES) good = barrier_wait(&sh.kv_empty[s], (n / STAGES - 1) & 1, &sh.broken);
                    if (!good) break;
                    barrier_expect(&sh.kv_full[s], kTileBytes<DP>);
                    load_tile<DP>(sh.kv[s], i == 0 ? &maps.k : &maps.v, kh, t * kTile, b, &sh.kv_full[s]);
                }
            }
            if (!good) {
                // copies under way write to this block's memory: it stays until they are done
                barrier_drain(&sh.q_full, 0);
                for (int i = n > STAGES ? n - STAGES : 0; i < n; ++i) barrier_drain(&sh.kv_full[i % STAGES], (i / STAGES) & 1);
            }
        }
        __syncwarp();
    } else if (warp == 17) {
        // ---- products
        if (elected()) {
            const int steps = (p.d + 15) / 16;
            const uint32_t score_kind = product_kind<T>(kTile, false), value_kind = product_kind<T>(steps * 16, true);
            const uint64_t query[2] = {channel_operand(shared_address(sh.q[0])), channel_operand(shared_address(sh.q[1]))};
            const uint64_t keys = channel_operand(shared_address(sh.kv[0])), values_at = row_operand(shared_address(sh.kv[0]));
            int used[2] = {0, 0}, n = 0;            // tiles that each query tile has taken; buffers
            bool last[2] = {false, false};          // which saw the tile before
            int last_v = 0;
            bool good = barrier_wait(&sh.q_full, 0, &sh.broken);
            // O += P V of the tile before, for query tile w
            const auto values = [&](int w) {
                if (!last[w] || !good) return;
                good = barrier_wait(&sh.p_full[w], (used[w] - 1) & 1, &sh.broken);
                if (!good) return;
                tmem_after();
                if (!*static_cast<volatile int *>(&sh.by_hand[w])) {
                    const uint64_t v = values_at + static_cast<uint32_t>(last_v * (kTileBytes<DP> >> 4));
                    const uint32_t out = tmem + 256 + w * kTile, prob = tmem + w * kTile;
                    const bool add = used[w] > 1;
#pragma unroll
                    for (int s = 0; s < kTile / 16; ++s) product_ts(out, prob + 8 * s + (s >= 4 ? 32 : 0), tile_rows(v, s), value_kind, add || s > 0);
                }
            };
            for (int t = t_begin; t < t_end && good; ++t) {
                const bool now[2] = {seen(0, t), seen(1, t)};
                if (!now[0] && !now[1]) continue;
                const int k = n % STAGES, v = (n + 1) % STAGES;
                const uint64_t key = keys + static_cast<uint32_t>(k * (kTileBytes<DP> >> 4));
                good = barrier_wait(&sh.kv_full[k], (n / STAGES) & 1, &sh.broken);
                // the values of the tile before have landed
                if (n > 0 && good) good = barrier_wait(&sh.kv_full[last_v], ((n - 1) / STAGES) & 1, &sh.broken);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    values(w);
                    if (!now[w] || !good) continue;
                    const uint32_t scores = tmem + w * kTile;
#pragma unroll
                    for (int s = 0; s < DP / 16; ++s)
                        if (s < steps) product_ss(scores, tile_channels(query[w], s), tile_channels(key, s), score_kind, s > 0);
                    products_done(&sh.s_full[w]);
                    ++used[w];
                }
                if (!good) break;
                if (n > 0) products_done(&sh.kv_empty[last_v]);
                products_done(&sh.kv_empty[k]);
                last[0] = now[0], last[1] = now[1];
                last_v = v;
                n += 2;
            }
            if (good && n > 0) good = barrier_wait(&sh.kv_full[last_v], ((n - 1) / STAGES) & 1, &sh.broken);
            for (int w = 0; w < 2; ++w) {
                if (good) values(w);
                products_done(&sh.o_full[w]);
            }
            if (!good) {
                barrier_drain(&sh.o_full[0], 0);
                barrier_drain(&sh.o_full[1], 0);
            }
        }
        __syncwarp();
    } else {
        // ---- softmax
        const int w = warp >> 3, half = warp >> 2 & 1, row = tid & 127, n = n0 + w * kTile + row;
        const uint32_t mine = tmem + (static_cast<uint32_t>(warp & 3) << 21);        // lanes 32 (warp mod 4) on
        const uint32_t scores = mine + w * kTile + half * 64, out = mine + 256 + w * kTile;
        const float factor = p.scale * kLog2e;
        const float inverse_cap = CAP ? p.scale / p.cap : 0.0f, outer = p.cap * kLog2e;
        const int doc = p.q_docs && n < p.N ? p.q_docs[static_cast<long long>(b) * p.N + n] : -1;
        const int limit = p.q_docs && doc < 0 ? 0 : key_limit(mask, n);
        const float slope = BIAS != kNoBias ? p.slopes[head] * kLog2e : 0.0f;
        const float2 here = BIAS != kNoBias ? map_place(n + mask.shift, p.width) : make_float2(0.0f, 0.0f);
        float ref = -INFINITY, sum = 0.0f, weight = 0.0f;       // sums of the probabilities, and of what they are rounded to
        int used = 0, buffers = 0, looks = 0;
        bool good = true;
        for (int t = t_begin; t < t_end; ++t) {
            const int other = state(1 - w, t), now = state(w, t);
            if (now == kHidden) {
                if (other != kHidden) buffers += 2;
                continue;
            }
            const int j0 = t * kTile + half * 64;
#pragma unroll
            for (int e = lane; e < 64; e += 32) {
                if (BIAS == kMapBias) {
                    const float2 at = map_place(j0 + e, p.width);
                    reinterpret_cast<float *>(sh.across[warp])[e] = at.x;
                    reinterpret_cast<float *>(sh.down[warp])[e] = at.y;
                }
                if (p.q_docs && now == kPartial)
                    reinterpret_cast<int *>(sh.docs[warp])[e] = j0 + e < p.M ? p.k_docs[static_cast<long long>(b) * p.M + j0 + e] : -1;
            }
            __syncwarp();
            good = good && barrier_wait(&sh.s_full[w], used & 1, &sh.broken);
            if (!good) break;
            tmem_after();
            // Probabilities of the thread's 64 scores for a reference, in registers; the largest score in units of log2.
            uint32_t packed[32];
            float part[2];
            const auto probabilities = [&](float base) {
                float high[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                Pair total(0.0f, 0.0f);
                const Pair by(GENERAL ? 1.0f : factor, GENERAL ? 1.0f : factor), less(-base, -base);
#pragma unroll
                for (int c = 0; c < 64; c += 32) {
                    uint32_t raw[32];
                    float *x = reinterpret_cast<float *>(raw);
                    tmem_load32(scores + c, raw);
                    tmem_loaded32(raw);
                    if constexpr (CAP) tanh_all<32>(x, inverse_cap);
                    if constexpr (GENERAL) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] *= CAP ? outer : factor;
                    }
                    if constexpr (BIAS == kMapBias) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 across = sh.across[warp][(c + i) / 4], down = sh.down[warp][(c + i) / 4];
#pragma unroll
                            for (int u = 0; u < 4; ++u)
                                x[i + u] = fmaf(-slope, fabsf(here.x - element(across, u)) + fabsf(here.y - element(down, u)), x[i + u]);
                        }
                    } else if constexpr (BIAS == kSequenceBias) {
                        const float from = here.y - static_cast<float>(j0 + c);
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = fmaf(-slope, fabsf(from - static_cast<float>(i)), x[i]);
                    }
                    if (now == kPartial) {
                        const int left = limit - j0 - c;
                        if (p.q_docs) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                const int4 id = sh.docs[warp][(c + i) / 4];
#pragma unroll
                                for (int u = 0; u < 4; ++u)
                                    if (i + u >= left || element(id, u) != doc) x[i + u] = -INFINITY;
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (i >= left) x[i] = -INFINITY;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        high[i % 4] = fmaxf(high[i % 4], x[i]);
                        high[i % 4 + 1] = fmaxf(high[i % 4 + 1], x[i + 1]);
                        const Pair at(x[i], x[i + 1]);
                        float e0, e1;
                        (GENERAL ? pair_add(at, less) : pair_fma(at, by, less)).get(e0, e1);
                        e0 = exp2_fast(e0);
                        e1 = exp2_fast(e1);
                        total = pair_add(total, Pair(e0, e1));
                        packed[(c + i) / 2] = pack_two<T>(e0, e1);
                    }
                }
                total.get(part[0], part[1]);
                const float most = fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3]));
                return GENERAL ? most : most * factor;
            };
            float high = probabilities((ref == -INFINITY ? 0.0f : ref) - held);
            // the two halves of a row agree on its largest score
            sh.high[used & 1][w][half][row] = high;
            warp_arrive(&sh.agreed[w][warp & 3]);
            good = barrier_wait(&sh.agreed[w][warp & 3], used & 1, &sh.broken);
            high = fmaxf(high, sh.high[used & 1][w][half ^ 1][row]);
            const bool grown = high > ref + slack;
            if (__any_sync(0xffffffffu, grown)) {
                // (a row that has seen nothing so far has zeros in O and sum: any factor does)
                const float shrink = grown ? (ref == -INFINITY ? 0.0f : exp2_fast(ref - high)) : 1.0f;
                ref = grown ? high : ref;
                sum *= shrink;
                weight *= shrink;
                if (used > 0) {
#pragma unroll 1
                    for (int c = half * (DP / 2); c < (half + 1) * (DP / 2); c += 32) {
                        uint32_t o[32];
                        tmem_load32(out + c, o);
                        tmem_loaded32(o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * shrink);
                        tmem_store32(out + c, o);
                    }
                }
                probabilities((ref == -INFINITY ? 0.0f : ref) - held);
            }
            tmem_store32(scores, packed);
            sum += part[0] + part[1];
            if (p.low) {
                Pair rounded(0.0f, 0.0f);
#pragma unroll
                for (int i = 0; i < 32; ++i) rounded = pair_add(rounded, Pair(DT<T>::unpack(packed[i], 0), DT<T>::unpack(packed[i], 1)));
                rounded.get(part[0], part[1]);
                weight += part[0] + part[1];
            }
            tmem_stored();
            bool hand = false;
            if (now == kPartial) {
                const int s = (buffers + 1) % STAGES;
                good = barrier_wait(&sh.kv_full[s], ((buffers + 1) / STAGES) & 1, &sh.broken);
                if (good && row_tainted<T, DP>(sh.kv[s], row, half)) *static_cast<volatile int *>(&sh.odd[w][looks % 3]) = 1;
                // (the slot after this one was last read two looks ago)
                if (row == 0 && half == 0) *static_cast<volatile int *>(&sh.odd[w][(looks + 1) % 3]) = 0;
                tmem_before();
                warp_arrive(&sh.looked[w]);
                good = good && barrier_wait(&sh.looked[w], looks & 1, &sh.broken);
                tmem_after();
                hand = __any_sync(0xffffffffu, good && *static_cast<volatile int *>(&sh.odd[w][looks % 3]) != 0);
                ++looks;
                if (hand && half == 0) {
                    const int *ids = p.k_docs ? p.k_docs + static_cast<long long>(b) * p.M + t * kTile : nullptr;
                    add_rows<T, DP, 64>(out, scores, sh.kv[s], used > 0, SeenRows{0, limit - t * kTile, ids, doc});
                }
            }
            if (row == 0 && half == 0) sh.by_hand[w] = hand;
            tmem_before();
            warp_arrive(&sh.p_full[w]);
            ++used;
            buffers += 2;
        }
        // the sum of the row's halves
        sh.high[used & 1][w][half][row] = sum;
        sh.weight[w][half][row] = weight;
        warp_arrive(&sh.agreed[w][warp & 3]);
        good = good && barrier_wait(&sh.agreed[w][warp & 3], used & 1, &sh.broken);
        sum += sh.high[used & 1][w][half ^ 1][row];
        weight += sh.weight[w][half ^ 1][row];
        if (good) good = barrier_wait(&sh.o_full[w], 0, &sh.broken);
        tmem_after();
        const bool empty = sum == 0.0f;
        const float inv = !good ? NAN : empty ? 0.0f : 1.0f / (p.low ? weight : sum);
        if (n0 + w * kTile < p.N && w < tiles) {          // whole warps
            const long long line = (static_cast<long long>(b) * p.h + head) * p.N + n;
            const long long part = static_cast<long long>(split) * p.B * p.h * p.N + line;
            const float lse = ref + log2f(sum) - held;
            if (n < p.N && half == 0) {
                if (p.splits > 1) p.part_lse[part] = empty ? -INFINITY : lse;
                else if (p.lse) p.lse[line] = empty ? INFINITY : lse;
            }
#pragma unroll 1
            for (int c = half * 32; c < DP && c < p.d; c += 64) {
                uint32_t o[32];
                if (used > 0) {
                    tmem_load32(out + c, o);
                    tmem_loaded32(o);
                }
                float y[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) y[i] = empty && good ? 0.0f : __uint_as_float(o[i]) * inv;
                if (n >= p.N) {
                    // no such query
                } else if (p.splits > 1) {
                    float *to = p.part_out + part * p.d + c;
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        if (c + i < p.d) *reinterpret_cast<float4 *>(to + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                } else {
                    const long long to = ((static_cast<long long>(b) * p.N + n) * p.h + head) * p.d + c;
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        if (c + i < p.d) {
                            store_eight<T>(static_cast<T *>(p.out) + to + i, y + i);
                            if (p.low) {
                                float rest[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) rest[e] = y[i + e] - DT<T>::rnd(y[i + e]);
                                store_eight<T>(static_cast<T *>(p.low) + to + i, rest);
                            }
                        }
                    }
                }
                __syncwarp();
            }
        }
    }
    tmem_before();
    __syncthreads();
    if (warp == 17) tmem_give(tmem);
}

template <typename T, int DP, bool CAP, GlobalBias BIAS>
cudaError_t forward_one(const GlobalParams &p, const GlobalMaps &maps, cudaStream_t stream)
{
    constexpr size_t smem = sizeof(ForwardShared<DP>) + 1024;
    static_assert(smem <= 227 * 1024 && smem > 114 * 1024, "one block per SM: it takes all of the tensor memory");
    const auto kernel = global_forward_kernel<T, DP, CAP, BIAS>;
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (err != cudaSuccess) return err;
    const dim3 grid(static_cast<unsigned>(p.B) * p.h * p.splits * ((p.N + p.block_rows - 1) / p.block_rows));
    return launch_chained(kernel, grid, kForwardThreads, smem, stream, p, maps);
}

}  // namespace

template <typename T>
cudaError_t run_global_forward(const GlobalParams &p, const GlobalMaps &maps, cudaStream_t stream)
{
    return by_scores(p, [&](auto width, auto cap, auto bias) {
        return forward_one<T, decltype(width)::value, decltype(cap)::value, decltype(bias)::value>(p, maps, stream);
    });
}

template cudaError_t run_global_forward<MATCHATTN_T>(const GlobalParams &, const GlobalMaps &, cudaStream_t);

}  // namespace matchattn
