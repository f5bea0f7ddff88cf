// Attention of drafted nodes over a paged KV cache — gfx950, f16 MFMA: a batch of sequences, a tree (or chain) of query rows each.
//
//   out[b, i, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(cap(scale * q[b, i, h] . k_j)),
//   j over the sequence's cached tokens (those of the row's window) and the drafted nodes that masks[b, i] names.
//
// All rows of a sequence share its cached tokens, so a workgroup owns one KV head of one sequence, up to 32 * CG (row, head-in-group) pairs,
// and one split of the tokens.  A wave holds 32 pairs as the columns of 32x32x16 matrix tiles; CG waves hold other pairs of the same tokens,
// the 4 / CG groups of such waves take every other 32 tokens of the split.  Per step the workgroup converts 32 tokens a group once into LDS as
// f16 (Q8g64 codes stay integers, exact, their scales beside them), and every wave runs
//   S^T[token, pair]  = sum_g k_scale_g[token] * (Kcodes_g . Q'^T)         Q' = q * 2^n of the pair, |Q'| < 2^9: exact for 16-bit queries
//   online softmax per pair (a pair is a lane and its partner 32 lanes on)
//   O^T[dim, pair]   += Vcodes^T . P'_g,   P'_g = p * v_scale_g as f16
// P' stays inside f16's range for any scale a cache can hold: the exponent of the largest V scale met so far is subtracted from the softmax
// reference, accumulators and sum carry it and it cancels.  What f16 cannot hold below its normal range is 2^-31 of the largest value met: a row
// whose own tokens' V scales all lie 2^20 and more below those of tokens that it gives no weight keeps fewer bits of its output, never of the sum of its
// probabilities (kSumLag; the vote for it costs under 1 %).
// MODE 0, 16-bit queries and bf16 outputs: the V rows of cached tokens are scaled once in LDS, f16(code * scale), and P is one f16.  Both
// roundings are 2^-11 of a value, a quarter of the output's own 2^-8 together; against f16 outputs (2^-11) they would be 1.6 times as far from 64 bits as an
// f32 attention rounded once (measured 3.2e-4 and 2.0e-4, 2-norm).  MODE 1, 16-bit queries and other outputs: codes exact, what f16 drops of P' as a
// second term.  MODE 2, f32 queries: what f16 drops of Q' too.
// Splits leave (partial, maximum, sum) records for gqa_draft_merge.
//
// What bounds it (times of calls in a row, with the merge).  64 rows of 64 / 8 heads of 128 on 50,000 tokens, 163-169 us: of a SIMD's ~ 360 K cycles
// vector instructions take 168 K and matrix instructions 100 K, of the CU's LDS its reads and writes 232 K; the two waves a SIMD that the registers
// allow overlap these in part.  Eight sequences of 5 rows (64 / 8) at 32,768 tokens, 160-164 us: 3.4 TB/s, vector instructions 45 %.  Eight ragged
// trees of up to 24 rows (32 / 8), 122-124 us.
// What carried it, in order (us of this kernel alone, chains / ragged trees / the wide tree, each in the build it was measured in): V scales folded and
// requests two steps ahead 430 / 531 / 524 -> 236 / 176 / 227; loads without
// conditions, which the compiler counts exactly, and nothing waiting for scales or table entries -> 210 / 149 / 194; operands read from LDS a phase
// ahead -> 187 / 134 / 185; queries formed under the first loads, groups of waves meeting in LDS, requests at a step's end -> 155 / 124 / 177.
#include <type_traits>

#include "gqa_prefill_x32.hpp"

namespace zllm {

namespace {

constexpr unsigned int kDraftThreads = 256;
constexpr float kValueBias = 14.0f; // of p times V scale: f16 ends at 2^16
// A folded tile's probabilities are summed as f16 holds them, in steps of 2^(lag - 31) where the tile's largest V scale lies 2^lag below the largest met: up to this
// lag, 2^-30 a token at most.  The sum does not have V's magnitude in it, so tiles further below are summed before they are rounded.
constexpr int kSumLag = 2;
constexpr float kFarScore = 16777216.0f; // f32 rounds what is larger by more than a half
// the exponents (biased) that a window of V scales may have: their powers of two, times the bias and a sum, stay inside f32
constexpr unsigned int kLeastExponent = 32u, kMostExponent = 247u;

// Places in LDS.  A row of K takes 16 bytes more than its values: a matrix operand's read, sixteen rows of one 16-byte chunk at a time, then meets
// every bank once, and every chunk is an immediate from one address.  A row of V takes no more (two workgroups have to fit a CU), the
// transposed read of four rows of 64 bytes meets every bank once because a row's 64-byte blocks change places by the row's low bits.
template <int D> constexpr int kKRow = D * 2 + 16;
template <int D> __device__ __forceinline__ unsigned int v_block_swap(unsigned int row)
{
    return D % 128 == 0 ? row & 3u : row >> 1 & 1u;
}

// A sequence's tokens and how they are cut: [first, end) = cached tokens some row's window reaches and the nodes that are there, in `parts`
// parts of `span` tokens (a multiple of 32).  No node: no part.
struct DraftSpan {
    unsigned int kv_len, count, first, end, parts, span;
};

__device__ __forceinline__ DraftSpan draft_span(const GqaDraftParams& p, unsigned int b)
{
    DraftSpan s;
    s.kv_len = min(p.kv_lens[b], kDraftMaxTokens);
    s.count = p.row_counts != nullptr ? min(p.row_counts[b], p.rows) : p.rows;
    s.first = p.window != 0u && s.kv_len + 1u > p.window ? s.kv_len + 1u - p.window : 0u;
    s.end = s.kv_len + s.count;
    const unsigned int tokens = s.end - s.first;
    s.parts = s.count == 0u ? 0u : min(p.max_chunks, (tokens + p.chunk_tokens - 1u) / p.chunk_tokens);
    s.span = s.parts == 0u ? 0u : ((tokens + s.parts - 1u) / s.parts + 31u) & ~31u;
    return s;
}

// The largest of a half of a wave, in all of its lanes: rows of sixteen by rotation, then the half's two rows
__device__ __forceinline__ float half_wave_max(float v)
{
    v = fmaxf(v, __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), 0x128, 0xf, 0xf, false)));
    v = fmaxf(v, __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), 0x124, 0xf, 0xf, false)));
    v = fmaxf(v, __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), 0x122, 0xf, 0xf, false)));
    v = fmaxf(v, __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), 0x121, 0xf, 0xf, false)));
    const u32x2_swap rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(rows.x), __uint_as_float(rows.y));
}

// Workgroups that a compute unit holds at once: what the launch bounds ask for, and what the plan of a call counts with
constexpr unsigned int groups_per_cu(unsigned int head_dim, unsigned int wave_columns, int mode)
{
    return head_dim <= 128u && wave_columns >= 2u && mode != 2 ? (head_dim == 64u ? 3u : 2u) : 1u;
}

// How an instantiation runs.  groups_per_cu: two where registers and LDS allow (one: 155 -> 215, 124 -> 202, 177 -> 239 us for
// the calls above), three at D 64 (two: 17 trees of 59, 32 / 8, at 5,584 tokens 177 -> 183; four spill: 191).  kTiles: tiles of 32 tokens a wave
// takes a step, two with four column waves, which have no token groups (one: 128 -> 143, 178 -> 196; D 192, 15 trees of up to 48 of 24 / 4 heads, 143 ->
// 158).  kAhead: matrix operands read a phase before they are needed, where registers are left for them (D 192 without: 137 -> 143; D 256, 36
// trees of 9 of 16 / 2 at 12,621 tokens 247 -> 260; f16 outputs at D 256, 7 trees of 19 at 20,085 tokens, 200 -> 223).
template <int D, bool F16, int CG, int MODE> struct DraftShape {
    static constexpr int kGroups = 4 / CG; // groups of waves, each with its own tokens
    static constexpr int kTiles = CG == 4 && MODE != 2 ? 2 : 1;
    static constexpr int kStepTiles = kGroups * kTiles;
    static constexpr int kUnits = D * (F16 ? 2 : 1) / 64; // 16-byte loads a thread, per 32 tokens of K and V
    static constexpr bool kAhead = MODE == 0 || (MODE == 1 && D > 128);
};

// SCALE32: the cache's scales have 32 bits, else 16.
template <int D, bool F16, int CG, int MODE, bool SCALE32>
__global__ __launch_bounds__(256, (groups_per_cu(D, CG, MODE))) void gqa_draft_partial(GqaDraftParams p)
{
    using Shape = DraftShape<D, F16, CG, MODE>;
    constexpr int TG = Shape::kGroups, NT = Shape::kTiles, TT = Shape::kStepTiles;
    constexpr bool EXACT = MODE != 0;          // probabilities in two terms
    constexpr bool QLO = MODE == 2;            // queries too
    constexpr bool FOLD = !F16 && !EXACT;      // V tiles of cached tokens are scaled in LDS
    constexpr int G = F16 ? 1 : D / 64;        // scale groups
    constexpr int KS = (F16 ? D : 64) / 16;    // matrix instructions a scale group takes per 32 tokens
    constexpr int DT = D / 32;
    constexpr int kRow = D * 2;
    constexpr int kRowUnits = D * (F16 ? 2 : 1) / 16; // 16-byte loads a row
    constexpr int kPlaneUnits = 32 * kRowUnits;
    constexpr int NU = Shape::kUnits;
    static_assert(NU * 256 == 2 * kPlaneUnits, "the threads take the units of a tile in whole rounds");
    struct Scales { // of a step, four steps in a ring
        float ks[TT][G][32];
        float vs[TT][G][32];          // of tiles that are not folded
        unsigned int fold[TT][G][32]; // of folded tiles: f16(scale * 2^(7 - exponent)), twice
        int exponent[TT];             // of the largest V scale of the tile, clamped
    };
    struct Lds {
        Scales scales[F16 ? 1 : 4];
        unsigned long long rows[4][TT * 32];
        // f16 rows off the main loop: a bit per V value that is no number (a zero stands in its place), and one more than the last step that has any
        unsigned char odd[2][F16 ? TT : 1][F16 ? 32 : 1][F16 ? D / 8 : 4];
        unsigned int odd_step[2][F16 ? TT : 1];
        __align__(16) unsigned char k[2][TT][32 * kKRow<D>];
        __align__(16) unsigned char v[2][TT][32 * kRow];
    };
    __shared__ __align__(16) Lds lds;

    const unsigned int tid = threadIdx.x;
    const unsigned int lane = tid & 63u;
    const unsigned int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned int cg = wave % CG;
    const unsigned int tg = wave / CG;
    const unsigned int n = lane & 31u; // column of a tile / row of an operand
    const unsigned int h = lane >> 5;

    // KV head fastest (with eight of them an XCD reads one), then the tiles of pairs of the same tokens, then the items
    const unsigned int kvh = blockIdx.x % p.num_kv_heads;
    const unsigned int tile = blockIdx.x / p.num_kv_heads % p.pair_tiles;
    const unsigned int item = blockIdx.x / p.num_kv_heads / p.pair_tiles;

    // ---- the item's sequence and part: items are numbered over the live parts of the batch ------------------------
    unsigned int b = 0, part = item, base = 0;
    bool found = false;
    DraftSpan span = {0u, 0u, 0u, 0u, 0u, 0u};
    for (unsigned int b0 = 0; b0 < p.batch; b0 += 64u) {
        const DraftSpan its = draft_span(p, min(b0 + lane, p.batch - 1u));
        const unsigned int parts = b0 + lane < p.batch ? its.parts : 0u;
        unsigned int sum = parts; // inclusive prefix sum over the lanes
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const unsigned int below = (unsigned int)__shfl_up((int)sum, off);
            sum += lane >= (unsigned int)off ? below : 0u;
        }
        const unsigned long long owner = __ballot(item < base + sum);
        if (owner != 0ull) {
            const int at = __builtin_ctzll(owner);
            b = b0 + (unsigned int)at;
            base += (unsigned int)__shfl((int)sum, at) - (unsigned int)__shfl((int)parts, at);
            part = item - base;
            span = {(unsigned int)__builtin_amdgcn_readlane(its.kv_len, at), (unsigned int)__builtin_amdgcn_readlane(its.count, at),
                    (unsigned int)__builtin_amdgcn_readlane(its.first, at), (unsigned int)__builtin_amdgcn_readlane(its.end, at),
                    (unsigned int)__builtin_amdgcn_readlane(its.parts, at), (unsigned int)__builtin_amdgcn_readlane(its.span, at)};
            found = true;
            break;
        }
        base += (unsigned int)__shfl((int)sum, 63);
    }
    if (!found) {
        return;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    part = __builtin_amdgcn_readfirstlane(part);
    if (part == 0u && tid == 0u && kvh == 0u && tile == 0u) {
        p.first_items[b] = item;
    }
    const unsigned long long part_begin = span.first + (unsigned long long)part * span.span;
    const unsigned int begin = (unsigned int)min(part_begin, (unsigned long long)span.end);
    const unsigned int end = (unsigned int)min(part_begin + span.span, (unsigned long long)span.end);
    const unsigned int kv_len = span.kv_len;

    // ---- this wave's pairs and their queries ----------------------------------------------------------------------
    struct Pair {
        unsigned int row, head;
        bool valid;
        unsigned int query_row;
    };
    auto pair_of = [&](unsigned int l) __attribute__((always_inline)) -> Pair { // of a lane; formed again where it is needed off the main loop
        const unsigned int pair = tile * (32u * CG) + cg * 32u + (l & 31u);
        const unsigned int row = pair / p.group;
        const bool valid = row < span.count;
        return {row, kvh * p.group + (pair - row * p.group), valid, b * p.rows + (valid ? row : 0u)};
    };
    auto position_of = [&](unsigned int query_row) __attribute__((always_inline)) -> unsigned int { return p.window != 0u ? max(p.positions[query_row], kv_len) : kv_len; };
    // requested first, formed when the first codes are under way
    u32x4 q_raw[D / 16][QLO ? 2 : 1];
    const Pair mine = pair_of(lane);
    const bool wave_valid = __any(mine.valid);
    {
        const size_t at = ((size_t)mine.query_row * p.num_heads + mine.head) * D + h * 8u;
        if (QLO && p.q_dtype == 0) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                q_raw[ks][0] = *(const u32x4*)((const float*)p.q + at + ks * 16);
                q_raw[ks][QLO ? 1 : 0] = *(const u32x4*)((const float*)p.q + at + ks * 16 + 4);
            }
        } else {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
                q_raw[ks][0] = *(const u32x4*)((const unsigned short*)p.q + at + ks * 16);
            }
        }
    }
    Frag qf[D / 16];
    Frag ql[QLO ? D / 16 : 1];
    float q_fac = 0.0f;
    auto form_queries = [&]() __attribute__((always_inline)) {
        auto values = [&](int ks, float (&x)[8]) __attribute__((always_inline)) {
            if (QLO && p.q_dtype == 0) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = __uint_as_float(q_raw[ks][0][e]);
                    x[4 + e] = __uint_as_float(q_raw[ks][QLO ? 1 : 0][e]);
                }
            } else {
                widen8(q_raw[ks][0], p.q_dtype, x);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = mine.valid ? x[e] : 0.0f;
            }
        };
        float amax = 0.0f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            float x[8];
            values(ks, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                amax = fmaxf(amax, fabsf(x[e]));
            }
        }
        amax = halves_max(amax);
        const unsigned int q_exp = min(max((__float_as_uint(amax) >> 23) & 0xffu, 16u), 254u);
        const float q_mul = __uint_as_float((262u - q_exp) << 23); // 2^(127 + 8 - q_exp)
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            float x[8];
            values(ks, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x0 = x[2 * e] * q_mul, x1 = x[2 * e + 1] * q_mul;
                const unsigned int word = pack_f16_hw(x0, x1);
                qf[ks].u[e] = word;
                if constexpr (QLO) {
                    const f16x2 hi = __builtin_bit_cast(f16x2, word);
                    ql[ks].u[e] = pack_f16_hw(x0 - (float)hi[0], x1 - (float)hi[1]);
                }
            }
        }
        q_fac = ldexpf(1.0f, (int)q_exp - 135);
    };
    const bool softcap = p.softcap != 0.0f;
    // scaled scores in base-2 units; with a soft cap in natural units first
    float mult = 0.0f; // of the pair, with its query's power of two
    const float inv_cap = softcap ? 1.0f / p.softcap : 0.0f;
    const float cap_log2 = p.softcap * kLog2e;

    // cached tokens [lo, kv_len) are visible to the pair's row; nodes by its mask
    auto lowest_of = [&](unsigned int position) __attribute__((always_inline)) -> unsigned int {
        return p.window != 0u && position >= p.window ? min(position - p.window + 1u, kv_len) : 0u; // nodes go by their own positions
    };
    unsigned int seen_by_all = 0u; // every row of the workgroup sees the cached tokens from here on
    if (p.window != 0u) {
        for (unsigned int j = lane; j < 32u * CG; j += 64u) {
            const unsigned int row = (tile * (32u * CG) + j) / p.group;
            seen_by_all = max(seen_by_all, row < span.count ? lowest_of(position_of(b * p.rows + row)) : 0u);
        }
        seen_by_all = wave_max_u(seen_by_all);
    }

    // ---- staging ---------------------------------------------------------------------------------------------------
    const unsigned int* table = p.tables + (size_t)b * p.table_stride;
    const unsigned int k_row = p.num_kv_heads * D * (F16 ? 2u : 1u); // bytes of a cache row
    const unsigned int head_at = kvh * D * (F16 ? 2u : 1u);
    const unsigned int steps = (end - begin + TT * 32u - 1u) / (TT * 32u);
    const unsigned int main_steps = end <= kv_len ? steps : (max(kv_len, begin) - begin) / (TT * 32u); // of cached tokens alone
    // `lead` of those hold tokens in front of some row's window.  A tile's V scales are taken as a whole where every row sees all of its tokens, so these steps take their
    // turn among the ones with nodes, behind the other cached tokens: visit v < main_visits is step v + lead.  (A loop of their own before the others spills up to 112
    // registers.  Five trees of 94 of 64 / 8 heads under a window of 1,024 68.8 -> 70.5 us, 16 of 8 of 32 / 8 24.4 -> 26.1, without a window no change.)
    const unsigned int lead = seen_by_all > begin ? min(main_steps, (seen_by_all - begin + TT * 32u - 1u) / (TT * 32u)) : 0u;
    const unsigned int main_visits = main_steps - lead;
    auto first_token = [&](unsigned int visit) __attribute__((always_inline)) -> unsigned int {
        const unsigned int step = visit >= main_steps ? visit : (visit >= main_visits ? visit - main_visits : visit + lead);
        return begin + step * (TT * 32u);
    };
    // Physical row of a token, in two steps: nothing is formed from a block-table entry before it is needed.  Tokens past the part repeat its last one.
    struct Place {
        unsigned int entry, offset;
    };
    auto look_up = [&](unsigned int token) __attribute__((always_inline)) -> Place {
        token = min(token, end - 1u);
        if (p.ring_capacity != 0u) {
            token %= p.ring_capacity;
        }
        const unsigned int page = p.block_shift < 32u ? token >> p.block_shift : token / p.block_tokens;
        return {table[min(page, p.table_stride - 1u)], token - page * p.block_tokens};
    };
    auto bytes_of = [&](const Place& place) __attribute__((always_inline)) -> unsigned long long { // to the row, in a plane of codes or f16 values
        return ((unsigned long long)place.entry * p.block_tokens + place.offset) * k_row;
    };
    // whether the thread's unit j of a tile is V's: known at compile time but where a round of the threads spans both planes
    auto in_v = [&](int j) __attribute__((always_inline)) -> bool {
        return 256 * j >= kPlaneUnits || (256 * (j + 1) > kPlaneUnits && tid + 256u * j >= (unsigned int)kPlaneUnits);
    };
    auto load_codes = [&](u32x4 (&raw)[TT][NU], unsigned int step) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
#pragma unroll
            for (int j = 0; j < NU; ++j) {
                const unsigned int unit = tid + 256u * j;
                const bool is_v = in_v(j);
                const unsigned int at = is_v ? unit - kPlaneUnits : unit;
                const unsigned long long row_at = lds.rows[step & 3u][t * 32 + at / kRowUnits];
                raw[t][j] = *(const u32x4*)((is_v ? p.v_plane : p.k_plane) + row_at + (head_at + at % kRowUnits * 16u));
            }
        }
    };
    // Wave w: the 64 scale rows of tile w % TT, K in the lower half; as they are stored
    auto load_scales = [&](unsigned int (&raw)[G], unsigned int step) __attribute__((always_inline)) {
        if constexpr (!F16) {
            const unsigned long long row_at = lds.rows[step & 3u][wave % TT * 32u + n] >> (SCALE32 ? 4 : 5); // 64 codes, one scale
            const unsigned char* from = (h != 0u ? p.v_scales : p.k_scales) + row_at + kvh * G * (SCALE32 ? 4u : 2u);
            if constexpr (SCALE32 || G % 2 == 0) { // words: two 16-bit scales each
#pragma unroll
                for (int w = 0; w < (SCALE32 ? G : G / 2); ++w) {
                    raw[w] = ((const unsigned int*)from)[w];
                }
            } else { // each on its own: two loads made one would be taken apart, and waited for, at once
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    raw[g] = __hip_atomic_load((const unsigned short*)from + g, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SINGLETHREAD);
                }
            }
        }
    };
    auto store_scales = [&](const unsigned int (&bits)[G], unsigned int step) __attribute__((always_inline)) {
        if constexpr (!F16) {
            if (wave < TT) {
                float raw[G];
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    if constexpr (SCALE32) {
                        raw[g] = __uint_as_float(bits[g]);
                    } else {
                        const unsigned short stored = (unsigned short)(G % 2 == 0 ? bits[g / 2] >> (16 * (g & 1)) : bits[g]);
                        raw[g] = p.scale_dtype == 1 ? f16_bits_to_f32(stored) : bf16_bits_to_f32(stored);
                    }
                }
                Scales& to = lds.scales[step & 3u];
                float top = 0.0f;
                bool odd = false;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const bool number = fabsf(raw[g]) < __builtin_inff();
                    odd = odd || !number;
                    top = fmaxf(top, number ? fabsf(raw[g]) : 0.0f);
                }
                top = half_wave_max(top);
                const int exponent = (int)min(max((__float_as_uint(top) >> 23) & 0xffu, kLeastExponent), kMostExponent);
                const float down = __uint_as_float((unsigned int)(127 + 7 + 127 - exponent) << 23);
                // a scale that is no number, of the K or the V row: the token's scores are none either
                const u32x2_swap either = __builtin_amdgcn_permlane32_swap((unsigned int)odd, (unsigned int)odd, false, false);
                odd = (either.x | either.y) != 0u;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    if (h == 0u) {
                        to.ks[wave][g][n] = odd ? __builtin_nanf("") : raw[g];
                    } else {
                        const float scale = odd ? 0.0f : raw[g];
                        to.vs[wave][g][n] = scale;
                        if constexpr (FOLD) {
                            to.fold[wave][g][n] = pack_f16_hw(scale * down, scale * down);
                        }
                    }
                }
                if (lane == 32u) {
                    to.exponent[wave] = exponent;
                }
            }
        }
    };
    // fold: a step of the main loop
    auto store_codes = [&](const u32x4 (&raw)[TT][NU], unsigned int buf, unsigned int step, bool fold) __attribute__((always_inline)) {
        unsigned int v_scales[FOLD ? TT : 1][FOLD ? NU : 1]; // all of them before the codes are waited for
        if constexpr (FOLD) {
            if (fold) {
#pragma unroll
                for (int t = 0; t < TT; ++t) {
#pragma unroll
                    for (int j = 0; j < NU; ++j) {
                        const unsigned int unit = tid + 256u * j;
                        const unsigned int at = in_v(j) ? unit - kPlaneUnits : 0u;
                        if (256u * j + 255u >= kPlaneUnits) {
                            v_scales[t][j] = lds.scales[step & 3u].fold[t][at % kRowUnits / 4u][at / kRowUnits];
                        }
                    }
                }
            }
            PREFILL_PHASE_FENCE();
        }
#pragma unroll
        for (int t = 0; t < TT; ++t) {
#pragma unroll
            for (int j = 0; j < NU; ++j) {
                const unsigned int unit = tid + 256u * j;
                const bool is_v = in_v(j);
                const unsigned int at = is_v ? unit - kPlaneUnits : unit;
                const unsigned int r = at / kRowUnits, c = at % kRowUnits;
                constexpr unsigned int kWide = F16 ? 16u : 32u; // bytes a unit takes in LDS
                unsigned char* to = is_v ? &lds.v[buf][t][r * kRow + ((c * kWide) ^ (v_block_swap<D>(r) << 6))] : &lds.k[buf][t][r * kKRow<D> + c * kWide];
                if constexpr (F16) {
                    u32x4 word = raw[t][j];
                    if (is_v && !fold) {
                        unsigned int odd = 0u;
#pragma unroll
                        for (int w = 0; w < 4; ++w) { // an exponent of ones carries into the sign
                            odd |= (word[w] & 0x7c007c00u) + 0x04000400u;
                        }
                        odd &= 0x80008000u;
                        if (odd != 0u) {
                            odd = 0u;
#pragma unroll
                            for (int w = 0; w < 4; ++w) {
                                const unsigned int bad = ((word[w] & 0x7c007c00u) + 0x04000400u) >> 15 & 0x00010001u;
                                word[w] &= ~(bad * 0xffffu);
                                odd |= ((bad | bad >> 15) & 3u) << (2 * w);
                            }
                            lds.odd_step[buf][t] = step + 1u;
                        }
                        lds.odd[buf][t][r][c] = (unsigned char)odd;
                    }
                    *(u32x4*)to = word;
                } else {
                    u32x4 half[2];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        unsigned int w0, w1;
                        codes4_to_f16(raw[t][j][w], w0, w1);
                        half[w >> 1][2 * (w & 1)] = w0, half[w >> 1][2 * (w & 1) + 1] = w1;
                    }
                    if (FOLD && is_v && fold) {
                        const f16x2 scale = __builtin_bit_cast(f16x2, v_scales[FOLD ? t : 0][FOLD ? j : 0]);
#pragma unroll
                        for (int w = 0; w < 8; ++w) {
                            const unsigned int word = half[w >> 2][w & 3];
                            half[w >> 2][w & 3] = __builtin_bit_cast(unsigned int, __builtin_bit_cast(f16x2, word) * scale);
                        }
                    }
                    *(u32x4*)to = half[0];
                    *(u32x4*)(to + 16) = half[1];
                }
            }
        }
    };

    f32x16 acc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            acc[t][i] = 0.0f;
        }
    }
    // acc and run_sum carry 2^(kValueBias - exponent of the largest V scale that the pair has met) (f16 rows: 2^kPBias)
    float run_max = kNegInf, run_sum = 0.0f;
    int window = (int)kLeastExponent; // that exponent, biased as f32's
    bool far_scores = false; // of the wave: a pair's run_max lies past kFarScore

    // Operand t, kk of a V tile: dims 32 t + lane % 32, tokens 16 kk + 4 h + {0 .. 3, 8 .. 11}, which are the tokens of elements 8 kk .. of the scores
    auto v_operand = [&](const unsigned char* vt, unsigned int l, int t, int kk) __attribute__((always_inline)) -> f16x8 {
        const unsigned int r = 4u * (l >> 5) + ((l & 15u) >> 2);
        const unsigned int at = r * kRow + ((unsigned int)(t * 64) ^ (v_block_swap<D>(r) << 6)) + (l >> 4 & 1u) * 32u + (l & 3u) * 8u;
        union {
            s16x4 s[2];
            f16x8 h;
        } vf;
        vf.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(vt + at + kk * 16 * kRow));
        vf.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4 __attribute__((address_space(3)))*)(vt + at + kk * 16 * kRow + 8 * kRow));
        return vf.h;
    };

    // Operands of a tile in registers: what the matrix instructions of the main loop take is read from LDS a phase earlier
    constexpr bool AHEAD = Shape::kAhead;
    auto k_operand = [&](const unsigned char* kt, unsigned int l, int ks) __attribute__((always_inline)) -> u32x4 {
        return *(const u32x4*)(kt + (l & 31u) * kKRow<D> + (l >> 5) * 16u + ks * 32);
    };
    constexpr int kFirstK = D / 32, kFirstV = (DT + 1) / 2; // half of them: the other half is read under the first one's matrix instructions
    auto read_k = [&](Frag (&kf)[AHEAD ? kFirstK : 1], unsigned int buf, unsigned int tt) __attribute__((always_inline)) {
        if constexpr (AHEAD) {
#pragma unroll
            for (int ks = 0; ks < kFirstK; ++ks) {
                kf[ks].u = k_operand(lds.k[buf][tt], lane, ks);
            }
            PREFILL_PHASE_FENCE();
        }
    };
    // s[i]: the score of token 8 (i / 4) + 4 h + i % 4 of tile tt, times 1 / mult
    auto scores = [&](auto tail, unsigned int buf, unsigned int step, unsigned int tt, const Frag (&kf)[AHEAD ? kFirstK : 1], f32x16& s) __attribute__((always_inline)) {
        constexpr bool TAIL = decltype(tail)::value;
        const unsigned int l = TAIL ? fresh_lane() : lane, h = l >> 5, m = l & 15u; // a tail's addresses take no registers of the main loop
        const unsigned char* kt = lds.k[buf][tt];
        const Scales& scales = lds.scales[F16 ? 0 : step & 3u];
        Frag rest[AHEAD ? kFirstK : 1];
        if constexpr (AHEAD && !TAIL) {
#pragma unroll
            for (int ks = 0; ks < kFirstK; ++ks) {
                rest[ks].u = k_operand(kt, l, kFirstK + ks);
            }
            PREFILL_PHASE_FENCE();
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
            f32x16 d;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                d[i] = 0.0f;
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                Frag k;
                if (AHEAD && !TAIL) {
                    k = g * KS + ks < kFirstK ? kf[(g * KS + ks) % (AHEAD ? kFirstK : 1)] : rest[(g * KS + ks) % (AHEAD ? kFirstK : 1)];
                } else {
                    k.u = k_operand(kt, l, g * KS + ks);
                }
                if constexpr (QLO) {
                    d = __builtin_amdgcn_mfma_f32_32x32x16_f16(k.h, ql[g * KS + ks].h, d, 0, 0, 0);
                }
                d = __builtin_amdgcn_mfma_f32_32x32x16_f16(k.h, qf[g * KS + ks].h, d, 0, 0, 0);
            }
            if constexpr (F16) {
                s = d;
            } else {
                // element i's token is the lane's row's lane i
                const float scale = scales.ks[tt][g][8u * (m >> 2) + 4u * h + (m & 3u)];
                if (g == 0) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[i] = row_lane(scale, i) * d[i];
                    }
                } else {
                    const float settled = d[0] * mult; // the compiler has waited for the matrix instruction here
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float t[4] = {s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]};
                        row_lane_fmac4(t[0], t[1], t[2], t[3], scale, q, d[4 * q], d[4 * q + 1], d[4 * q + 2], d[4 * q + 3], settled);
                        s[4 * q] = t[0], s[4 * q + 1] = t[1], s[4 * q + 2] = t[2], s[4 * q + 3] = t[3];
                    }
                }
            }
        }
    };
    // Rows that see a token with V values that are no numbers have none in those dimensions, and zeros in their place keep them from the rows that do not (a weight of
    // zero does not: zero times infinity).  Looking for them costs the f16 window case (4 x 12 rows, 16 / 8 heads of 256, a few steps a workgroup) 22.7 -> 24.0 us.
    auto mark_odd = [&](unsigned int buf, unsigned int tt, unsigned int seen) __attribute__((always_inline)) {
        if constexpr (F16) {
            const unsigned int h = fresh_lane() >> 5;
            const unsigned int half = (seen & 0x0f0f0f0fu) << (4u * h), tokens = half | (unsigned int)__shfl_xor((int)half, 32);
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                unsigned int hit = 0u; // a bit per dim of the tile
#pragma unroll 1
                for (unsigned int token = 0; token < 32u; ++token) {
                    hit |= (tokens >> token & 1u) != 0u ? *(const unsigned int*)&lds.odd[buf][F16 ? tt : 0u][F16 ? token : 0u][t * 4] : 0u;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    acc[t][i] = hit >> (8u * (i >> 2) + 4u * h + (i & 3)) & 1u ? __builtin_nanf("") : acc[t][i];
                }
            }
        }
    };
    // TAIL: the tile holds drafted nodes, tokens in front of a window, or ends with the part; else every row sees all of its tokens, those past the part aside
    auto attend = [&](auto tail, unsigned int buf, unsigned int step, unsigned int tt, unsigned int t0, int tile_exponent, f32x16& s, auto between) __attribute__((always_inline)) {
        constexpr bool TAIL = decltype(tail)::value;
        const unsigned int l = TAIL ? fresh_lane() : lane, h = l >> 5;
        constexpr bool PLAIN = F16 && !EXACT;
        constexpr bool FOLDED = FOLD && !TAIL;
        const unsigned char* vt = lds.v[buf][tt];
        const Scales& scales = lds.scales[F16 ? 0 : step & 3u];
        f16x8 vf[AHEAD && !TAIL ? kFirstV : 1][2];
        if constexpr (AHEAD && !TAIL) {
#pragma unroll
            for (int t = 0; t < kFirstV; ++t) {
                vf[t][0] = v_operand(vt, l, t, 0);
                vf[t][1] = v_operand(vt, l, t, 1);
            }
            PREFILL_PHASE_FENCE();
        }
        // ---- softmax; `fac`: what is left to multiply the scores with
        float fac = mult;
        if (softcap) {
            asm volatile(""); // a branch: without it both sides are computed and chosen from
            fac = 1.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float y = s[i] * mult * inv_cap;
                // a score that is no number stays one; past f32's range the power is infinite, its reciprocal zero
                s[i] = EXACT ? (y == y ? cap_log2 * soft_tanh(y) : y)
                             : cap_log2 * fmaf(-2.0f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(y * (2.0f * kLog2e)) + 1.0f), 1.0f);
            }
        }
        unsigned int seen = ~0u; // TAIL: bit 8 (i / 4) + i % 4 for element i
        if constexpr (TAIL) {
            const Pair own = pair_of(l);
            const unsigned int position = position_of(own.query_row), lo = lowest_of(position);
            const int first_node = (int)(t0 - kv_len); // below zero where cached tokens lead
            if (p.masks != nullptr) {
                const unsigned long long* words = p.masks + (size_t)own.query_row * p.mask_words;
                const unsigned int base = (unsigned int)max(first_node, 0), word = min(base >> 6, p.mask_words - 1u), shift = base & 63u;
                const unsigned long long low = words[word], high = words[min(word + 1u, p.mask_words - 1u)];
                seen = (unsigned int)(low >> shift | (shift > 32u && word + 1u < p.mask_words ? high << (64u - shift) : 0ull));
                if (first_node <= -32) {
                    seen = ~0u;
                } else if (first_node < 0) {
                    seen = seen << -first_node | ((1u << -first_node) - 1u);
                }
            } else {
                const int nodes = (int)own.row - first_node + 1;
                seen = nodes >= 32 ? ~0u : (nodes <= 0 ? 0u : (1u << nodes) - 1u);
            }
            seen &= end - t0 < 32u ? (1u << (end - t0)) - 1u : ~0u;
            seen &= lo <= t0 ? ~0u : (lo - t0 < 32u ? ~0u << (lo - t0) : 0u);
            seen = own.valid ? seen >> (4u * h) : 0u;
            if (p.window != 0u) {
                unsigned int at[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int node = first_node + 8 * (i >> 2) + (int)(4u * h) + (i & 3);
                    at[i] = p.positions[(size_t)b * p.rows + (unsigned int)min(max(node, 0), (int)p.rows - 1)];
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int node = first_node + 8 * (i >> 2) + (int)(4u * h) + (i & 3);
                    const unsigned int its = max(at[i], kv_len); // positions may be the largest there are: no sums
                    const bool near = node < 0 || its >= position || position - its < p.window;
                    seen &= near ? ~0u : ~(1u << (8 * (i >> 2) + (i & 3)));
                }
            }
            if constexpr (F16) {
                if (__builtin_amdgcn_readfirstlane(lds.odd_step[buf][tt]) == step + 1u) {
                    mark_odd(buf, tt, seen);
                }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = seen >> (8 * (i >> 2) + (i & 3)) & 1u ? s[i] : kNegInf;
            }
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) {
            top = fmaxf(top, s[i]);
        }
        top *= fac;
        // the window of V scales: of the tile, or of the tokens that the pair sees (others may hold anything)
        int now = window, exponent = window;
        if constexpr (!F16) {
            if constexpr (!TAIL) {
                exponent = __builtin_amdgcn_readfirstlane(tile_exponent);
            } else {
                float scale_top = 0.0f;
#pragma unroll
                for (int g = 0; g < G; ++g) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float scale = scales.vs[tt][g][8 * (i >> 2) + 4 * h + (i & 3)];
                        scale_top = fmaxf(scale_top, (seen >> (8 * (i >> 2) + (i & 3)) & 1u) != 0u ? fabsf(scale) : 0.0f);
                    }
                }
                scale_top = halves_max(scale_top);
                exponent = (int)min(max((__float_as_uint(scale_top) >> 23) & 0xffu, kLeastExponent), kMostExponent);
            }
            now = max(window, exponent);
        }
        // A reference stays while no score passes it by more than kSlack powers of two: f16 holds p of up to 2^13 here.  Measured against the tile's own maximum where
        // scales follow in the product.
        if (__any((FOLDED || PLAIN ? top - run_max > kSlack : top > run_max) || now != window)) {
            const float new_max = fmaxf(run_max, halves_max(top));
            const float keep = __builtin_amdgcn_exp2f(run_max - (new_max == kNegInf ? 0.0f : new_max));
            const float alpha = ldexpf(keep, window - now);
            run_sum = ldexpf(run_sum * keep, window - now); // 2^(window - now) alone may lie below f32's range
            run_max = new_max;
            window = now;
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                acc[t] *= alpha;
            }
            far_scores = __any(fabsf(run_max) > kFarScore && run_max != kNegInf);
        }
        float reference = run_max == kNegInf ? 0.0f : run_max;
        // The reference is a rounded product, and what it is subtracted from in a multiply-add is not: far from zero what its rounding left is more than a power of two, and p
        // would leave f16.  Such pairs' scores are rounded first.
        if (far_scores) {
            const bool far = fabsf(reference) > kFarScore;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float rounded = s[i] * fac;
                asm volatile("" : "+v"(rounded)); // no multiply-add
                s[i] = far ? rounded - reference : s[i];
            }
            fac = far ? 1.0f : fac;
            reference = far ? 0.0f : reference;
        }
        float pr[16];
        if constexpr (FOLDED || PLAIN) {
            // p of a folded tile carries 2^(7 + its exponent - the window), so that p . V' carries what acc carries
            const int lag = FOLDED ? window - exponent : 0;
            const bool far = FOLDED && __any(lag > kSumLag);
            const float shift = FOLDED ? (float)(far ? 7 : 7 - lag) - reference : kPBias - reference;
            Frag ph[2];
            float sum = 0.0f, exact = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                pr[i] = __builtin_amdgcn_exp2f(fmaf(s[i], fac, shift));
            }
            if (far) {
                asm volatile(""); // a branch
                const float down = ldexpf(1.0f, -lag);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    exact += pr[i];
                    pr[i] *= down;
                }
            }
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                const unsigned int word = pack_f16_hw(pr[i], pr[i + 1]);
                ph[i >> 3].u[(i & 7) >> 1] = word;
                sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, word), f16x2{(_Float16)1.0f, (_Float16)1.0f}, sum, false); // what is multiplied is what is summed
            }
            between();
            run_sum = FOLDED ? fmaf(far ? exact : sum, __uint_as_float((unsigned int)(127 + 7 + 127 - (far ? window : exponent)) << 23), run_sum) : run_sum + sum;
#pragma unroll
            for (int t = 0; t < DT; ++t) {
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    f16x8 v;
                    if (AHEAD && !TAIL && t < kFirstV) {
                        v = vf[t % (AHEAD && !TAIL ? kFirstV : 1)][kk];
                    } else {
                        v = v_operand(vt, l, t, kk);
                    }
                    acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[kk].h, acc[t], 0, 0, 0);
                }
            }
        } else {
            const float shift = (F16 ? kPBias : kValueBias + (float)(127 - window)) - reference;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                pr[i] = __builtin_amdgcn_exp2f(fmaf(s[i], fac, shift));
                sum += pr[i];
            }
            between();
            run_sum += sum;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                Frag ph[2], pl[2];
                const float v_scale = F16 ? 0.0f : scales.vs[tt][g][8u * (l >> 2 & 3u) + 4u * h + (l & 3u)]; // element i's token is the lane's row's lane i
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        f32x4 x = {pr[8 * kk + 4 * q], pr[8 * kk + 4 * q + 1], pr[8 * kk + 4 * q + 2], pr[8 * kk + 4 * q + 3]};
                        if constexpr (!F16) {
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                x[r] = row_lane(v_scale, 8 * kk + 4 * q + r) * x[r];
                            }
                        }
                        ph[kk].u[2 * q] = pack_f16_hw(x[0], x[1]);
                        ph[kk].u[2 * q + 1] = pack_f16_hw(x[2], x[3]);
                        if constexpr (EXACT) {
                            const f16x2 h0 = __builtin_bit_cast(f16x2, pack_f16_hw(x[0], x[1])), h1 = __builtin_bit_cast(f16x2, pack_f16_hw(x[2], x[3]));
                            pl[kk].u[2 * q] = pack_f16_hw(x[0] - (float)h0[0], x[1] - (float)h0[1]);
                            pl[kk].u[2 * q + 1] = pack_f16_hw(x[2] - (float)h1[0], x[3] - (float)h1[1]);
                        }
                    }
                }
#pragma unroll
                for (int t = g * (DT / G); t < (g + 1) * (DT / G); ++t) {
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk) {
                        const f16x8 v = AHEAD && !TAIL && t < kFirstV ? vf[t % (AHEAD && !TAIL ? kFirstV : 1)][kk] : v_operand(vt, l, t, kk);
                        if constexpr (EXACT) {
                            acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[kk].h, acc[t], 0, 0, 0);
                        }
                        acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[kk].h, acc[t], 0, 0, 0);
                    }
                }
            }
        }
    };

    // ---- the part's tokens.  A step ends with the next step's codes and the scales of the one after it going to LDS (a folded tile needs its
    // scales a step before its codes), and with what the steps after those need being requested: loads are under way for a whole step.  All
    // requests go on past the last step, on the part's last row: without conditions the compiler counts the loads in flight and waits for none
    // too early.
    if (steps != 0u) {
        Place ahead;
        unsigned int scale_raw[G];
        u32x4 raw[TT][NU];
        const unsigned int slot = tid % (TT * 32u);
        {
            Place places[4];
#pragma unroll
            for (unsigned int step = 0; step < 4u; ++step) {
                places[step] = look_up(first_token(step) + slot);
            }
            ahead = look_up(first_token(4u) + slot);
#pragma unroll
            for (unsigned int step = 0; step < 4u; ++step) {
                lds.rows[step][slot] = bytes_of(places[step]);
            }
        }
        __syncthreads();
        if (F16 && tid < 2u * TT) {
            lds.odd_step[tid / TT][F16 ? tid % TT : 0u] = 0u;
        }
        {
            unsigned int first[2][G];
            load_scales(first[0], 0);
            load_scales(first[1], 1);
            load_codes(raw, 0);
            load_scales(scale_raw, 2);
            form_queries();
            mult = softcap ? q_fac * p.score_scale : q_fac * p.score_scale * kLog2e;
            store_scales(first[0], 0);
            store_scales(first[1], 1);
        }
        __syncthreads();
        store_codes(raw, 0, 0, main_visits != 0u);
        load_codes(raw, 1);
        __syncthreads();
        auto turn = [&](unsigned int buf, unsigned int step) __attribute__((always_inline)) {
            if (step + 1u < steps) {
                store_codes(raw, buf ^ 1u, step + 1u, step + 1u < main_visits);
            }
            load_codes(raw, step + 2u);
            if (step + 2u < steps) {
                store_scales(scale_raw, step + 2u);
            }
            load_scales(scale_raw, step + 3u);
            lds.rows[step & 3u][slot] = bytes_of(ahead);
            ahead = look_up(first_token(step + 5u) + slot);
            __syncthreads();
        };
        auto body = [&](auto parity, unsigned int step) __attribute__((always_inline)) {
            constexpr unsigned int BUF = decltype(parity)::value;
            const unsigned int t0 = begin + (step + lead) * (TT * 32u) + tg * (NT * 32u);
            if (wave_valid && t0 < end) {
                Frag kf[AHEAD ? kFirstK : 1];
                int exponents[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    exponents[j] = F16 ? 0 : lds.scales[F16 ? 0 : step & 3u].exponent[tg * NT + j];
                }
                read_k(kf, BUF, tg * NT);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if (j == 0 || t0 + j * 32u < end) {
                        f32x16 s;
                        scores(std::false_type{}, BUF, step, tg * NT + j, kf, s);
                        attend(std::false_type{}, BUF, step, tg * NT + j, t0 + j * 32u, exponents[j], s, [&]() __attribute__((always_inline)) {
                            if (j + 1 < NT) {
                                PREFILL_PHASE_FENCE();
                                read_k(kf, BUF, tg * NT + j + 1);
                            }
                        });
                    }
                }
            }
            turn(BUF, step);
        };
        unsigned int step = 0;
        for (; step + 1u < main_visits; step += 2u) {
            body(std::integral_constant<unsigned int, 0>{}, step);
            body(std::integral_constant<unsigned int, 1>{}, step + 1u);
        }
        if (step < main_visits) {
            body(std::integral_constant<unsigned int, 0>{}, step);
            ++step;
        }
        // the steps with drafted nodes, and those in front of a window, a tile at a time through one piece of code
        for (; step < steps; ++step) {
#pragma unroll 1
            for (int j = 0; j < NT; ++j) {
                const unsigned int t0 = first_token(step) + (tg * NT + j) * 32u;
                if (wave_valid && t0 < end) {
                    f32x16 s;
                    Frag none[AHEAD ? kFirstK : 1];
                    scores(std::true_type{}, step & 1u, step, tg * NT + j, none, s);
                    attend(std::true_type{}, step & 1u, step, tg * NT + j, t0, 0, s, []() {});
                }
            }
            turn(step & 1u, step);
        }
    }

    // ---- the record, in true units; the groups of waves that had other tokens of the same pairs meet in LDS first -------------------------
    const unsigned int last_lane = fresh_lane();
    float total = halves_sum(run_sum);
    {
        const int down = F16 ? -(int)kPBias : window - 127 - (int)kValueBias;
        const float fa = ldexpf(1.0f, down / 2), fb = ldexpf(1.0f, down - down / 2); // two factors: 2^down alone may leave f32's range
        total *= fa;
        total *= fb;
        run_max = total == 0.0f ? kNegInf : run_max;
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            acc[t] *= fa;
            acc[t] *= fb;
        }
    }
    if constexpr (TG > 1) {
        struct Shares {
            f32x4 acc[TG - 1][CG][DT * 4][64];
            f32x2 stats[TG - 1][CG][64];
        };
        static_assert(sizeof(Shares) <= sizeof(lds.k) + sizeof(lds.v), "the shares take the tiles' place");
        Shares& shares = *(Shares*)&lds.k[0][0][0];
        // the tiles are read no more: every wave has passed the barrier that ends the last step
        if (tg != 0u) {
#pragma unroll
            for (int t = 0; t < DT; ++t) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    shares.acc[tg - 1u][cg][t * 4 + q][last_lane] = f32x4{acc[t][4 * q], acc[t][4 * q + 1], acc[t][4 * q + 2], acc[t][4 * q + 3]};
                }
            }
            shares.stats[tg - 1u][cg][last_lane] = f32x2{run_max, total};
        }
        __syncthreads();
        if (tg != 0u) {
            return;
        }
#pragma unroll
        for (int k = 0; k < TG - 1; ++k) {
            const f32x2 stat = shares.stats[k][cg][last_lane];
            const float all = fmaxf(run_max, stat[0]), safe = all == kNegInf ? 0.0f : all;
            const float mine_weight = __builtin_amdgcn_exp2f(run_max - safe), its_weight = __builtin_amdgcn_exp2f(stat[0] - safe);
            run_max = all;
            total = total * mine_weight + stat[1] * its_weight;
#pragma unroll
            for (int t = 0; t < DT; ++t) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 its = shares.acc[k][cg][t * 4 + q][last_lane];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        acc[t][4 * q + r] = fmaf(its[r], its_weight, acc[t][4 * q + r] * mine_weight);
                    }
                }
            }
        }
    }
    const Pair own = pair_of(last_lane);
    if (!own.valid) {
        return;
    }
    const size_t rec = ((size_t)item * p.rows + own.row) * p.num_heads + own.head;
    if (last_lane < 32u) {
        p.stats[rec * 2] = run_max;
        p.stats[rec * 2 + 1] = total;
    }
    float* out = p.partial + rec * (size_t)D + 4u * (last_lane >> 5);
#pragma unroll
    for (int t = 0; t < DT; ++t) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            *(f32x4*)(out + t * 32 + q * 8) = f32x4{acc[t][4 * q], acc[t][4 * q + 1], acc[t][4 * q + 2], acc[t][4 * q + 3]};
        }
    }
}

// out = sum_c partial_c 2^(max_c - M) / sum_c sum_c 2^(max_c - M), zeros for rows that are not there and rows that see nothing.  D / 4 threads take
// four dims each of every SPREADth record of a (row, head), four records' loads at a time, and the SPREAD shares meet in LDS: a wait for
// memory is 1 us, and a call of few rows has many records for each (7 rows of 16 heads with 68 records, one thread after the other: 60 us).
template <int D, int SPREAD> __global__ __launch_bounds__(256) void gqa_draft_merge(GqaDraftParams p)
{
    constexpr unsigned int kQuads = D / 4;
    constexpr unsigned int kUnits = 256 / (kQuads * SPREAD);
    __shared__ __align__(16) f32x4 shares[SPREAD > 1 ? kUnits * SPREAD * kQuads : 1];
    __shared__ float share_stats[SPREAD > 1 ? kUnits * SPREAD : 1][2];
    const unsigned int quad = threadIdx.x % kQuads, share = threadIdx.x / kQuads % SPREAD, sub = threadIdx.x / (kQuads * SPREAD);
    const unsigned long long units = (unsigned long long)p.batch * p.rows * p.num_heads;
    const unsigned long long wanted = (unsigned long long)blockIdx.x * kUnits + sub;
    const bool there = sub < kUnits && wanted < units;
    const unsigned long long unit = there ? wanted : units - 1u;
    const unsigned int query_row = (unsigned int)(unit / p.num_heads);
    const unsigned int head = (unsigned int)(unit - (unsigned long long)query_row * p.num_heads);
    const unsigned int b = query_row / p.rows, row = query_row % p.rows;
    const unsigned int first = p.first_items[b];
    const DraftSpan span = draft_span(p, b);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    float total = 0.0f, top = kNegInf;
    if (there && row < span.count) {
        const unsigned int records = min(span.parts, p.items - min(first, p.items));
        const size_t stride = (size_t)p.rows * p.num_heads;
        const size_t rec0 = (size_t)first * stride + (size_t)row * p.num_heads + head;
        for (unsigned int c0 = share; c0 < records; c0 += 4u * SPREAD) {
            f32x2 stat[4];
            f32x4 part[4];
#pragma unroll
            for (unsigned int e = 0; e < 4u; ++e) { // past the last record: the first of the four again, with no weight
                const size_t rec = rec0 + (size_t)(c0 + e * SPREAD < records ? c0 + e * SPREAD : c0) * stride;
                stat[e] = *(const f32x2*)(p.stats + rec * 2);
                part[e] = *(const f32x4*)(p.partial + rec * D + quad * 4u);
            }
            float now = top;
#pragma unroll
            for (unsigned int e = 0; e < 4u; ++e) {
                now = fmaxf(now, stat[e][0]);
            }
            const float safe = now == kNegInf ? 0.0f : now;
            const float keep = __builtin_amdgcn_exp2f(top - safe);
            sum *= keep;
            total *= keep;
            top = now;
#pragma unroll
            for (unsigned int e = 0; e < 4u; ++e) {
                const float weight = c0 + e * SPREAD < records ? __builtin_amdgcn_exp2f(stat[e][0] - safe) : 0.0f;
                total = fmaf(weight, stat[e][1], total);
                sum += weight * part[e];
            }
        }
    }
    if constexpr (SPREAD > 1) {
        const unsigned int slot = sub * SPREAD + share;
        if (sub < kUnits) {
            shares[slot * kQuads + quad] = sum;
            if (quad == 0u) {
                share_stats[slot][0] = top;
                share_stats[slot][1] = total;
            }
        }
        __syncthreads();
        if (sub >= kUnits || share != 0u) {
            return;
        }
        float all = kNegInf;
#pragma unroll
        for (int k = 0; k < SPREAD; ++k) {
            all = fmaxf(all, share_stats[slot + k][0]);
        }
        const float safe = all == kNegInf ? 0.0f : all;
        sum = f32x4{0.f, 0.f, 0.f, 0.f};
        total = 0.0f;
#pragma unroll
        for (int k = 0; k < SPREAD; ++k) {
            const float weight = __builtin_amdgcn_exp2f(share_stats[slot + k][0] - safe);
            total = fmaf(weight, share_stats[slot + k][1], total);
            sum += weight * shares[(slot + k) * kQuads + quad];
        }
    }
    if (!there) {
        return;
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    f32x4 v = sum * inv;
    if (p.gate != nullptr && total != 0.0f) { // a row of zeros stays one, whatever its gate holds
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = gated(v[e], p.gate, p.gate_cols, p.gate_dtype, query_row, head * D + quad * 4u + e);
        }
    }
    const size_t at = unit * D + quad * 4u;
    if (p.out_dtype == 0) {
        *(f32x4*)((float*)p.out + at) = v;
    } else if (p.out_dtype == 1) {
        *(u32x2*)((unsigned short*)p.out + at) = u32x2{pack_bf16_hw(v[0], v[1]), pack_bf16_hw(v[2], v[3])};
    } else {
        *(u32x2*)((unsigned short*)p.out + at) = u32x2{pack_f16_hw(v[0], v[1]), pack_f16_hw(v[2], v[3])};
    }
}

template <int D, bool F16, bool SCALE32, int MODE> void launch_draft_mode(const GqaDraftParams& p, hipStream_t stream)
{
    const dim3 grid(p.items * p.pair_tiles * p.num_kv_heads), block(kDraftThreads);
    if (p.token_groups == 1u) {
        gqa_draft_partial<D, F16, 4, MODE, SCALE32><<<grid, block, 0, stream>>>(p);
    } else if (p.token_groups == 2u) {
        gqa_draft_partial<D, F16, 2, MODE, SCALE32><<<grid, block, 0, stream>>>(p);
    } else if constexpr (D <= 128) {
        gqa_draft_partial<D, F16, 1, MODE, SCALE32><<<grid, block, 0, stream>>>(p);
    }
}

template <int D, bool F16, bool SCALE32> void launch_draft_partial(const GqaDraftParams& p, hipStream_t stream)
{
    if (p.mode == 0) {
        launch_draft_mode<D, F16, SCALE32, 0>(p, stream);
    } else if (p.mode == 1) {
        launch_draft_mode<D, F16, SCALE32, 1>(p, stream);
    } else {
        gqa_draft_partial<D, F16, 2, 2, SCALE32><<<dim3(p.items * p.pair_tiles * p.num_kv_heads), dim3(kDraftThreads), 0, stream>>>(p);
    }
}

template <int D> void launch_draft_partial_q8(const GqaDraftParams& p, hipStream_t stream)
{
    if (p.scale_dtype == 2) {
        launch_draft_partial<D, false, true>(p, stream);
    } else {
        launch_draft_partial<D, false, false>(p, stream);
    }
}

// Shares where a thread alone would wait for memory too often and the device has room: 16 records and more, and fewer workgroups without shares than
// CUs.  Measured at D 128, eight shares against one: 256 units of 32 records 4.0 and 6.2 us, 512 of 61 5.0 and 10.5, 1,024 of 61 9.9 and 11,
// 1,536 of 32 6.7 and 7.1; but 2,048 of 32 9.9 and 7.6, 4,096 of 16 10.2 and 7.0, and 2,560 of 8, where three of a share's four loads repeat, 6.1 and 4.3.
template <int D> void launch_draft_merge(const GqaDraftParams& p, hipStream_t stream)
{
    constexpr unsigned int kAlone = 256 / (D / 4); // units of a workgroup without shares
    constexpr int kSpread = kAlone >= 8 ? 8 : 4;
    constexpr unsigned int kShared = 256 / (D / 4 * kSpread);
    const unsigned long long units = (unsigned long long)p.batch * p.rows * p.num_heads;
    const unsigned long long groups = gqa_draft_merge_groups(units, D);
    if (p.max_chunks >= 16u && groups < 256u) {
        gqa_draft_merge<D, kSpread><<<dim3((unsigned int)((units + kShared - 1u) / kShared)), dim3(256), 0, stream>>>(p);
    } else {
        gqa_draft_merge<D, 1><<<dim3((unsigned int)groups), dim3(256), 0, stream>>>(p);
    }
}

} // namespace

// Pairs fill as few waves as hold them; what is left of a workgroup's four waves takes other tokens.  28 pairs over 4,096 tokens in one column
// wave 12.1 us, in two 13.8; 40 pairs (the eight sequences above) in two 154, in four 177.  One column wave leaves the four token groups no room at
// head dimensions of 192 and more; f32 queries, two terms each, have registers for two groups' tiles only.
unsigned int gqa_draft_wave_columns(unsigned int pairs, unsigned int head_dim, int mode)
{
    if (mode == 2) {
        return 2u;
    }
    if (pairs <= 32u && head_dim <= 128u) {
        return 1u;
    }
    return pairs <= 64u ? 2u : 4u;
}

unsigned int gqa_draft_groups_per_cu(unsigned int head_dim, unsigned int wave_columns, int mode)
{
    return groups_per_cu(head_dim, wave_columns, mode);
}

unsigned long long gqa_draft_merge_groups(unsigned long long units, unsigned int head_dim)
{
    const unsigned int alone = 256u / (head_dim / 4u);
    return (units + alone - 1u) / alone;
}

hipError_t launch_gqa_draft_attention(const GqaDraftParams& p, int kv_format, hipStream_t stream)
{
    if (kv_format == 1) {
        switch (p.head_dim) {
        case 128: launch_draft_partial<128, true, false>(p, stream); break;
        default: launch_draft_partial<256, true, false>(p, stream); break;
        }
    } else {
        switch (p.head_dim) {
        case 64: launch_draft_partial_q8<64>(p, stream); break;
        case 128: launch_draft_partial_q8<128>(p, stream); break;
        case 192: launch_draft_partial_q8<192>(p, stream); break;
        default: launch_draft_partial_q8<256>(p, stream); break;
        }
    }
    hipError_t rc = hipGetLastError();
    if (rc != hipSuccess) {
        return rc;
    }
    switch (p.head_dim) {
    case 64: launch_draft_merge<64>(p, stream); break;
    case 128: launch_draft_merge<128>(p, stream); break;
    case 192: launch_draft_merge<192>(p, stream); break;
    default: launch_draft_merge<256>(p, stream); break;
    }
    return hipGetLastError();
}

} // namespace zllm
