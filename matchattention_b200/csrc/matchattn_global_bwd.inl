// Dense attention, backward, 16-bit types of up to 128 channels, on the matrix units.  Included once per type with MATCHATTN_T
// defined.
//
//   P = 2^(x - lse),  dP = dO V^T,  dS = P (1 - tanh^2) (dP - delta),  delta = rowsum(dO O)
//   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K
//
// Two passes of one kernel, each recomputing S and P: for keys (a block owns 128 keys of a key head, walks the queries of all
// heads that share it, and keeps dK and dV in tensor memory) and for queries (128 queries, walks the keys, keeps dQ).  That is seven
// products (one of them in two terms) where one pass with dQ added up in global memory has five, but the sums have one order and no atomics.
//
// A block has a fixed pair of tiles (keys: K, V; queries: Q, dO) and a moving pair (Q, dO; K, V).  The scores and dP of
// fixed by moving rows come to tensor memory; a thread holds a fixed row and 32 of the 128 moving ones (warps 0-15), and puts P over S
// and dS over dP, rounded to the type (which the matrix unit asks for), as first operands of the products that add up the moving rows.
// dQ takes dS as two terms, cut to the type and what that left, in two products: rounded once, its error beside those of delta and of the
// result made dQ 1.41 to 1.5 times as far from the exact gradient as the result's own rounding; it is 1.01 to 1.05 times now (dK and
// dV stand at 1.35 to 1.45 times), for 570 us in place of 526 in the second case below.  Order of the matrix unit: dV(i-1), S(i),
// dK(i-1), dP(i): while threads take exponentials of tile i it forms dK(i-1) and dP(i), while they form dS(i) it forms dV(i) and S(i+1).
//
// float16 has few exponents: P is held times 2^12 (P of a row of 10^5 tokens is not subnormal), dS times the power of two that
// brings the largest value that |dS| <= |dO| |V| + |delta| allows over the tiles that the block meets to between 2^14 and 2^15; both leave
// the sums exactly.  The bound knows only tokens of visible pairs (global_levels_kernel): what is hidden, another item, another key
// head, or a tile that the block never meets, however large, takes no digits from a sum.
//
// Measured, one B200: 2 x 4096 tokens, 16 heads x 128 on 4 key heads, bfloat16, causal and capped 345 us (dK, dV) and 322 us (dQ); 8160
// tokens, 8 heads x 16, float16, map bias 686 and 570.  Bound by the steps that a tile goes through one after another (scores, P,
// dP, dS); with eight warps of 64 rows each and the rows' figures fetched within the tile 497 + 407 and 843 + 650.
//
// As in the forward pass, tiles that are partly hidden are looked through for infinite and NaN values, and added term by term
// where they have some.
#include "matchattn_global_mma.cuh"

namespace matchattn {
namespace {

constexpr int kBackThreads = 576;
constexpr int kPart = 32;                // moving rows of a thread

template <int DP>
struct BackShared {
    static constexpr int kStages = DP == 128 ? 2 : 3;
    uint8_t fixed[2][kTileBytes<DP>];
    uint8_t moving[kStages][2][kTileBytes<DP>];
    float4 lse[16][8], delta[16][8], across[16][8], down[16][8];      // per warp, for its 32 moving rows; less delta; column and row on the map
    int4 docs[16][8];
    uint64_t fixed_full, full[kStages], empty[kStages], s_full, p_full, dp_full, ds_full, done, looked, stored;
    uint32_t tmem;
    int broken, by_hand[2], odd[2][3];
    float level[16];             // float16: what a warp has found of the bound of |dS|
    int begin[16];               // the tile's first moving row, for the rare path (a register less)
};

// KEYS: the pass for dK and dV
template <typename T, int DP, bool CAP, GlobalBias BIAS, bool KEYS>
__global__ void __launch_bounds__(kBackThreads, 1) global_backward_kernel(const GlobalParams p, const __grid_constant__ GlobalMaps maps)
{
    chain_begin();
    constexpr int STAGES = BackShared<DP>::kStages;
    constexpr bool HALF = std::is_same<T, __half>::value;
    constexpr float kLift = HALF ? 12.0f : 0.0f;           // log2 of the factor that P is held by
    extern __shared__ uint8_t raw_shared[];
    BackShared<DP> &sh = *reinterpret_cast<BackShared<DP> *>(raw_shared + (1024 - (shared_address(raw_shared) & 1023)) % 1024);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int heads = KEYS ? p.hk : p.h;
    const int each = p.B * heads, lot = KEYS ? each * p.head_splits : each;
    const int turn = blockIdx.x / lot, split = blockIdx.x % lot / each, b = blockIdx.x % each / heads, own = blockIdx.x % each % heads, kh = KEYS ? own : own / p.g;
    // causal: the first keys are seen by most queries, the last queries see most keys: their blocks begin first
    const int f0 = (KEYS ? turn : gridDim.x / lot - 1 - turn) * kTile;
    const GlobalMask mask = global_mask(p, b);
    const int key_tiles = (p.M + kTile - 1) / kTile, query_tiles = (p.N + kTile - 1) / kTile;
    const DocRange *kr = p.q_docs ? p.ranges + p.B * query_tiles + b * key_tiles : nullptr;
    const DocRange *qr = p.q_docs ? p.ranges + b * query_tiles : nullptr;
    const auto state = [&](int t) {
        const int n0 = KEYS ? t * kTile : f0, j0 = KEYS ? f0 : t * kTile;
        return tile_state(mask, p.N, n0, j0, qr ? qr + n0 / kTile : nullptr, kr ? kr + j0 / kTile : nullptr);
    };
    // heads that are walked
    const int r_begin = KEYS ? first_head(p, split) : 0, rounds = KEYS ? first_head(p, split + 1) : 1;
    const int t_begin = KEYS ? min(query_begin(mask, f0), p.N) / kTile : 0;
    const int t_end = KEYS ? query_tiles : (key_limit(mask, min(f0 + kTile, p.N) - 1) + kTile - 1) / kTile;

    if (HALF && warp < 16) {
        // the largest |dS| that the norms of the tiles allow
        float most = 0.0f;
        const int walk = t_end - t_begin;
        for (long long e = tid; e < static_cast<long long>(rounds - r_begin) * walk; e += 512) {
            const int r = r_begin + static_cast<int>(e / walk), t = t_begin + static_cast<int>(e % walk);
            if (state(t) == kHidden) continue;
            const long long query = (static_cast<long long>(b) * p.h + (KEYS ? kh * p.g + r : own)) * query_tiles + (KEYS ? t : f0 / kTile);
            const long long key = (static_cast<long long>(b) * p.hk + kh) * key_tiles + (KEYS ? f0 / kTile : t);
            most = fmaxf(most, fmaf(p.level_o[query], p.level_v[key], p.level_delta[query]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        if (lane == 0) sh.level[warp] = most;
    }
    if (tid == 0) {
        barrier_init(&sh.fixed_full, 1);
        for (int i = 0; i < STAGES; ++i) {
            barrier_init(&sh.full[i], 1);
            barrier_init(&sh.empty[i], 1);
        }
        barrier_init(&sh.s_full, 1);
        barrier_init(&sh.dp_full, 1);
        barrier_init(&sh.done, 1);
        barrier_init(&sh.p_full, 16);
        barrier_init(&sh.ds_full, 16);
        barrier_init(&sh.looked, 16);
        barrier_init(&sh.stored, 16);
        sh.broken = 0;
        for (int i = 0; i < 3; ++i) sh.odd[0][i] = sh.odd[1][i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 17) tmem_take(&sh.tmem);
    tmem_before();
    __syncthreads();
    tmem_after();
    const uint32_t tmem = sh.tmem;
    const uint32_t scores = tmem, slopes = tmem + 128, sum_v = tmem + 256, sum_k = tmem + 384;       // sum_k: dK or dQ

    if (warp == 16) {
        // ---- copies
        if (elected()) {
            barrier_expect(&sh.fixed_full, 2 * kTileBytes<DP>);
            load_tile<DP>(sh.fixed[0], KEYS ? &maps.k : &maps.q, own, f0, b, &sh.fixed_full);
            load_tile<DP>(sh.fixed[1], KEYS ? &maps.v : &maps.o, own, f0, b, &sh.fixed_full);
            int i = 0;
            bool good = true;
            for (int r = r_begin; r < rounds && good; ++r)
                for (int t = t_begin; t < t_end; ++t) {
                    if (state(t) == kHidden) continue;
                    const int s = i % STAGES, head = KEYS ? kh * p.g + r : kh;
                    if (i >= STAGES) good = barrier_wait(&sh.empty[s], (i / STAGES - 1) & 1, &sh.broken);
                    if (!good) break;
                    barrier_expect(&sh.full[s], 2 * kTileBytes<DP>);
                    load_tile<DP>(sh.moving[s][0], KEYS ? &maps.q : &maps.k, head, t * kTile, b, &sh.full[s]);
                    load_tile<DP>(sh.moving[s][1], KEYS ? &maps.o : &maps.v, head, t * kTile, b, &sh.full[s]);
                    ++i;
                }
            if (!good) {
                // copies under way write to this block's memory: it stays until they are done
                barrier_drain(&sh.fixed_full, 0);
                for (int n = i > STAGES ? i - STAGES : 0; n < i; ++n) barrier_drain(&sh.full[n % STAGES], (n / STAGES) & 1);
            }
        }
        __syncwarp();
    } else if (warp == 17) {
        // ---- products
        if (elected()) {
            const int steps = (p.d + 15) / 16;
            const uint32_t score_kind = product_kind<T>(kTile, false), sum_kind = product_kind<T>(steps * 16, true);
            const uint64_t fixed[2] = {channel_operand(shared_address(sh.fixed[0])), channel_operand(shared_address(sh.fixed[1]))};
            const uint64_t by_channel = channel_operand(shared_address(sh.moving[0][0])), by_row = row_operand(shared_address(sh.moving[0][0]));
            bool good = barrier_wait(&sh.fixed_full, 0, &sh.broken);
            int i = 0;
            const auto moving = [&](uint64_t first, int n, int which) {
                return first + static_cast<uint32_t>((n % STAGES * 2 + which) * (kTileBytes<DP> >> 4));
            };
            // columns of a first operand: 32 moving rows in the first 16 words of every 32
            const auto add_up = [&](uint32_t sums, uint32_t weights, uint64_t tile, bool add) {
#pragma unroll
                for (int s = 0; s < kTile / 16; ++s) product_ts(sums, weights + 32 * (s / 2) + 8 * (s % 2), tile_rows(tile, s), sum_kind, add || s > 0);
            };
            const auto scores_of = [&](uint32_t to, uint64_t a, uint64_t b) {
#pragma unroll
                for (int s = 0; s < DP / 16; ++s)
                    if (s < steps) product_ss(to, tile_channels(a, s), tile_channels(b, s), score_kind, s > 0);
            };
            const auto after_scores = [&](int n) {         // dV of tile n, when its P is there
                good = good && barrier_wait(&sh.p_full, n & 1, &sh.broken);
                if (!good) return;
                tmem_after();
                if (KEYS && !*static_cast<volatile int *>(&sh.by_hand[0])) add_up(sum_v, scores, moving(by_row, n, 1), n > 0);
            };
            const auto after_slopes = [&](int n) {         // dK or dQ of tile n, when its dS is there
                good = good && barrier_wait(&sh.ds_full, n & 1, &sh.broken);
                if (!good) return;
                tmem_after();
                if (!*static_cast<volatile int *>(&sh.by_hand[1])) {
                    add_up(sum_k, slopes, moving(by_row, n, 0), n > 0);
                    if (!KEYS) add_up(sum_k, slopes + 16, moving(by_row, n, 0), true);        // the second terms of dS
                }
                products_done(&sh.empty[n % STAGES]);
            };
            for (int r = r_begin; r < rounds && good; ++r)
                for (int t = t_begin; t < t_end && good; ++t) {
                    if (state(t) == kHidden) continue;
                    good = barrier_wait(&sh.full[i % STAGES], (i / STAGES) & 1, &sh.broken);
                    if (i > 0) after_scores(i - 1);
                    if (!good) break;
                    scores_of(scores, fixed[0], moving(by_channel, i, 0));
                    products_done(&sh.s_full);
                    if (i > 0) after_slopes(i - 1);
                    if (!good) break;
                    scores_of(slopes, fixed[1], moving(by_channel, i, 1));
                    products_done(&sh.dp_full);
                    ++i;
                }
            if (good && i > 0) {
                after_scores(i - 1);
                after_slopes(i - 1);
            }
            products_done(&sh.done);
            if (!good) barrier_drain(&sh.done, 0);
        }
        __syncwarp();
    } else {
        // ---- probabilities and slopes
        const int w = warp >> 2, f = f0 + (tid & 127);                          // quarter of the moving rows; the fixed row
        const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
        const uint32_t my_scores = scores + lanes + w * kPart, my_slopes = slopes + lanes + w * kPart;
        const float factor = p.scale * kLog2e, inverse_cap = CAP ? p.scale / p.cap : 0.0f, outer = p.cap * kLog2e;
        // dS is held times 2^(lift - kLift), the sums of dS times 2^-lift
        int lift = 0;
        if (HALF) {
            float bound = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) bound = fmaxf(bound, sh.level[e]);
            if (bound > 0.0f && bound <= 3.402823466e38f) lift = min(max(14 - ilogbf(bound), -60), 60);
        }
        const float hold = ldexpf(1.0f, lift) * (HALF ? 1.0f / 4096.0f : 1.0f);
        int doc = -1;
        if (p.q_docs) {
            if (KEYS) doc = f < p.M ? p.k_docs[static_cast<long long>(b) * p.M + f] : -1;
            else doc = f < p.N ? p.q_docs[static_cast<long long>(b) * p.N + f] : -1;
        }
        const bool apart = p.q_docs && doc < 0;                                 // of no document
        const int limit = apart ? 0 : key_limit(mask, f);                       // queries: keys below it are seen
        const int first = apart ? 1 << 30 : query_begin(mask, f);               // keys: queries from it on see it
        const float2 here = BIAS != kNoBias ? map_place(KEYS ? f : f + mask.shift, p.width) : make_float2(0.0f, 0.0f);
        float lse = INFINITY, delta = 0.0f;
        if (!KEYS && f < p.N) {
            const long long line = (static_cast<long long>(b) * p.h + own) * p.N + f;
            lse = p.lse[line] - kLift;
            delta = p.delta[line];
        }
        // what a lane fetches of a tile's moving rows, one row of the warp's 32; a tile ahead, because it takes as long as a tile
        float next_lse = 0.0f, next_delta = 0.0f;
        int next_doc = -1;
        const auto fetch = [&](int r, int t) {
            const int m = t * kTile + w * kPart + lane;
            if (KEYS) {
                const long long line = (static_cast<long long>(b) * p.h + kh * p.g + r) * p.N + m;
                next_lse = m < p.N ? p.lse[line] - kLift : INFINITY;
                next_delta = m < p.N ? p.delta[line] : 0.0f;
            }
            if (p.q_docs) {
                const int rows = KEYS ? p.N : p.M;
                next_doc = m < rows ? (KEYS ? p.q_docs : p.k_docs)[static_cast<long long>(b) * rows + m] : -1;
            }
        };
        // the visible tile after (r, t)
        const auto advance = [&](int &r, int &t) {
            do {
                if (++t >= t_end) t = t_begin, ++r;
            } while (r < rounds && state(t) == kHidden);
        };
        int i = 0, looks = 0, stores = 0, r = r_begin, t = t_begin - 1;
        bool good = true;
        if (t_begin < t_end) advance(r, t);
        else r = rounds;
        if (r < rounds) fetch(r, t);
        for (; r < rounds;) {
            {
                const int head = KEYS ? kh * p.g + r : own, now = state(t);
                const float slope = BIAS != kNoBias ? p.slopes[head] * kLog2e : 0.0f;
                const int m0 = t * kTile + w * kPart;                           // first of the warp's moving rows
                if (KEYS) {
                    reinterpret_cast<float *>(sh.lse[warp])[lane] = next_lse;
                    reinterpret_cast<float *>(sh.delta[warp])[lane] = -next_delta;
                }
                if (p.q_docs) reinterpret_cast<int *>(sh.docs[warp])[lane] = next_doc;
                if (lane == 0) sh.begin[warp] = t * kTile;
                if (BIAS == kMapBias) {
                    const float2 at = map_place(KEYS ? m0 + lane + mask.shift : m0 + lane, p.width);
                    reinterpret_cast<float *>(sh.across[warp])[lane] = at.x;
                    reinterpret_cast<float *>(sh.down[warp])[lane] = at.y;
                }
                __syncwarp();
                advance(r, t);
                if (r < rounds) fetch(r, t);
                good = good && barrier_wait(&sh.s_full, i & 1, &sh.broken);
                if (!good) break;
                tmem_after();
                float prob[kPart];                                              // P, then P (1 - tanh^2)
                uint32_t *raw = reinterpret_cast<uint32_t *>(prob);
                tmem_load32(my_scores, raw);
                tmem_loaded32(raw);
                const float from = here.y - static_cast<float>(KEYS ? m0 + mask.shift : m0);
                const int bar = (KEYS ? first : limit) - m0;                    // keys: the moving rows from it on are seen; queries: those below
                const auto seen_rows = [&] {
                    const int tile0 = sh.begin[warp];
                    const int *ids = KEYS ? p.q_docs : p.k_docs;
                    if (ids != nullptr) ids += static_cast<long long>(b) * (KEYS ? p.N : p.M) + tile0;
                    return KEYS ? SeenRows{first - tile0, p.N - tile0, ids, doc} : SeenRows{0, limit - tile0, ids, doc};
                };
                {
                    uint32_t packed[16];
                    if (CAP) tanh_all<32>(prob, inverse_cap);
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const int four = e / 4;
                        float level[4], value[4];
                        float4 row_lse, across, down;
                        int4 docs;
                        if (KEYS) row_lse = sh.lse[warp][four];
                        if (BIAS == kMapBias) across = sh.across[warp][four], down = sh.down[warp][four];
                        if (now == kPartial && p.q_docs) docs = sh.docs[warp][four];
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const int at = e + u;
                            level[u] = KEYS ? element(row_lse, u) : lse;
                            if (BIAS == kMapBias) level[u] = fmaf(slope, fabsf(here.x - element(across, u)) + fabsf(here.y - element(down, u)), level[u]);
                            if (BIAS == kSequenceBias) level[u] = fmaf(slope, fabsf(from - static_cast<float>(at)), level[u]);
                            float slant = 1.0f;
                            if (CAP) {
                                slant = fmaf(-prob[at], prob[at], 1.0f);
                                value[u] = fmaf(outer, prob[at], -level[u]);
                            } else {
                                value[u] = fmaf(prob[at], factor, -level[u]);
                            }
                            if (now == kPartial) {
                                bool seen = KEYS ? at >= bar : at < bar;
                                if (p.q_docs) seen = seen && element(docs, u) == doc;
                                if (!seen) value[u] = -INFINITY;
                            }
                            value[u] = exp2_fast(value[u]);
                            prob[at] = CAP ? value[u] * slant : value[u];
                        }
                        packed[e / 2] = pack_two<T>(value[0], value[1]);
                        packed[e / 2 + 1] = pack_two<T>(value[2], value[3]);
                    }
                    if (KEYS) tmem_store16(my_scores, packed);
                }
                if (KEYS) tmem_stored();
                // a partly hidden tile's moving rows are looked through: warps 0-7 the first tile, 8-15 the second
                bool hand_v = false, hand_k = false;
                if (now == kPartial) {
                    const int s = i % STAGES;
                    good = barrier_wait(&sh.full[s], (i / STAGES) & 1, &sh.broken);
                    if (good && (KEYS || w < 2) && row_tainted<T, DP>(sh.moving[s][w >> 1], tid & 127, w & 1))
                        *static_cast<volatile int *>(&sh.odd[w >> 1][looks % 3]) = 1;
                    // (the slot after this one was last read two looks ago)
                    if ((tid & 255) == 0) *static_cast<volatile int *>(&sh.odd[w >> 1][(looks + 1) % 3]) = 0;
                    tmem_before();
                    warp_arrive(&sh.looked);
                    good = good && barrier_wait(&sh.looked, looks & 1, &sh.broken);
                    tmem_after();
                    hand_k = __any_sync(0xffffffffu, good && *static_cast<volatile int *>(&sh.odd[0][looks % 3]) != 0);
                    hand_v = KEYS && __any_sync(0xffffffffu, good && *static_cast<volatile int *>(&sh.odd[1][looks % 3]) != 0);
                    ++looks;
                    if (hand_v && w == 0) add_rows<T, DP, kPart>(sum_v + lanes, scores + lanes, sh.moving[s][1], i > 0, seen_rows());
                }
                if (tid == 0) sh.by_hand[0] = hand_v;
                tmem_before();
                warp_arrive(&sh.p_full);
                good = good && barrier_wait(&sh.dp_full, i & 1, &sh.broken);
                if (!good) break;
                tmem_after();
                {
                    uint32_t dp[32], packed[KEYS ? 16 : 32];
                    tmem_load32(my_slopes, dp);
                    tmem_loaded32(dp);
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        float4 row_delta;
                        if (KEYS) row_delta = sh.delta[warp][e / 4];
                        float value[4];
#pragma unroll
                        for (int u = 0; u < 4; u += 2) {
                            Pair off = pair_add(Pair(__uint_as_float(dp[e + u]), __uint_as_float(dp[e + u + 1])),
                                                KEYS ? Pair(element(row_delta, u), element(row_delta, u + 1)) : Pair(-delta, -delta));
                            if (HALF) off = pair_mul(off, Pair(hold, hold));
                            pair_mul(Pair(prob[e + u], prob[e + u + 1]), off).get(value[u], value[u + 1]);
                        }
                        if (!KEYS) {
                            // cut to the digits of the type, and what that leaves
#pragma unroll
                            for (int u = 0; u < 4; u += 2) {
                                const Pair whole(value[u], value[u + 1]);
                                float rest[2];
                                value[u] = __uint_as_float(__float_as_uint(value[u]) & (HALF ? 0xffffe000u : 0xffff0000u));
                                value[u + 1] = __uint_as_float(__float_as_uint(value[u + 1]) & (HALF ? 0xffffe000u : 0xffff0000u));
                                pair_fma(Pair(value[u], value[u + 1]), Pair(-1.0f, -1.0f), whole).get(rest[0], rest[1]);
                                packed[16 + (e + u) / 2] = pack_two<T>(rest[0], rest[1]);
                            }
                        }
                        packed[e / 2] = pack_two<T>(value[0], value[1]);
                        packed[e / 2 + 1] = pack_two<T>(value[2], value[3]);
                    }
                    if (now == kPartial) {
                        // hidden pairs, whose figures may be NaN: zeros (in a loop of its own: within the one above it cost every tile 5 %)
                        const int begin = (KEYS ? first : limit) - sh.begin[warp] - w * kPart;
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            int4 docs;
                            if (p.q_docs) docs = sh.docs[warp][e / 4];
#pragma unroll
                            for (int u = 0; u < 4; ++u) {
                                const bool seen = (KEYS ? e + u >= begin : e + u < begin) && (!p.q_docs || element(docs, u) == doc);
                                if (!seen) {
                                    packed[(e + u) / 2] &= u & 1 ? 0x0000ffffu : 0xffff0000u;
                                    if (!KEYS) packed[16 + (e + u) / 2] &= u & 1 ? 0x0000ffffu : 0xffff0000u;
                                }
                            }
                        }
                    }
                    if (KEYS) tmem_store16(my_slopes, packed);
                    else tmem_store32(my_slopes, packed);
                }
                tmem_stored();
                if (hand_k) {
                    tmem_before();
                    warp_arrive(&sh.stored);
                    good = barrier_wait(&sh.stored, stores & 1, &sh.broken);
                    tmem_after();
                    ++stores;
                    if (w == 1) {
                        add_rows<T, DP, kPart>(sum_k + lanes, slopes + lanes, sh.moving[i % STAGES][0], i > 0, seen_rows());
                        if (!KEYS) add_rows<T, DP, kPart>(sum_k + lanes, slopes + 16 + lanes, sh.moving[i % STAGES][0], true, seen_rows());
                    }
                }
                if (tid == 0) sh.by_hand[1] = hand_k;
                tmem_before();
                warp_arrive(&sh.ds_full);
                ++i;
            }
        }
        if (good) good = barrier_wait(&sh.done, 0, &sh.broken);
        tmem_after();
        // ---- results: dV by warps 0-7 and dK by 8-15, or dQ by all, the channels in turn
        const int rows = KEYS ? p.M : p.N;
        const float times = KEYS && w < 2 ? (HALF ? 1.0f / 4096.0f : 1.0f) : p.scale * ldexpf(1.0f, -lift);
        T *to = static_cast<T *>(KEYS ? (w < 2 ? p.d_v : p.d_k) : p.d_q) + ((static_cast<long long>(b) * rows + f) * heads + own) * p.d;
        const uint32_t from = (KEYS && w < 2 ? sum_v : sum_k) + lanes;
#pragma unroll 1
        for (int c = 32 * (KEYS ? w & 1 : w); c < DP && c < p.d; c += KEYS ? 64 : 128) {
            uint32_t raw[32] = {};
            if (i > 0) {
                tmem_load32(from + c, raw);
                tmem_loaded32(raw);
            }
            if (f < rows) {
                float y[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) y[e] = good ? __uint_as_float(raw[e]) * times : NAN;
#pragma unroll
                for (int e = 0; e < 32; e += 8)
                    if (c + e < p.d) {
                        if (KEYS && p.head_splits > 1) {
                            float4 *part = reinterpret_cast<float4 *>((w < 2 ? p.part_v : p.part_k) +
                                                                      (((static_cast<long long>(split) * p.B + b) * rows + f) * heads + own) * p.d + c + e);
                            part[0] = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
                            part[1] = make_float4(y[e + 4], y[e + 5], y[e + 6], y[e + 7]);
                        } else {
                            store_eight<T>(to + c + e, y + e);
                        }
                    }
            }
            __syncwarp();
        }
    }
    tmem_before();
    __syncthreads();
    if (warp == 17) tmem_give(tmem);
}

template <typename T, int DP, bool CAP, GlobalBias BIAS, bool KEYS>
cudaError_t backward_pass(const GlobalParams &p, const GlobalMaps &maps, cudaStream_t stream)
{
    constexpr size_t smem = sizeof(BackShared<DP>) + 1024;
    static_assert(smem <= 227 * 1024 && smem > 114 * 1024, "one block per SM: it takes all of the tensor memory");
    const auto kernel = global_backward_kernel<T, DP, CAP, BIAS, KEYS>;
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (err != cudaSuccess) return err;
    const dim3 grid(static_cast<unsigned>(p.B) * (KEYS ? p.hk * p.head_splits : p.h) * (((KEYS ? p.M : p.N) + kTile - 1) / kTile));
    return launch_chained(kernel, grid, kBackThreads, smem, stream, p, maps);
}

}  // namespace

template <typename T>
cudaError_t run_global_backward(const GlobalParams &p, const GlobalMaps &maps, cudaStream_t stream)
{
    return by_scores(p, [&](auto width, auto cap, auto bias) {
        constexpr int DP = decltype(width)::value;
        constexpr bool CAP = decltype(cap)::value;
        constexpr GlobalBias BIAS = decltype(bias)::value;
        const cudaError_t err = backward_pass<T, DP, CAP, BIAS, true>(p, maps, stream);
        return err != cudaSuccess ? err : backward_pass<T, DP, CAP, BIAS, false>(p, maps, stream);
    });
}

template cudaError_t run_global_backward<MATCHATTN_T>(const GlobalParams &, const GlobalMaps &, cudaStream_t);

}  // namespace matchattn
