// Attention over a layer's paged KV cache (include/kvsnap_attention.h).
//
// With scores s_t = scale q.k_t over the tokens a row sees, out = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m) for any m;
// the kernels go over the tokens once with m the largest score so far, scaling what they hold when it grows, so no
// score is kept.  Parts of a row's tokens are joined the same way: each part gives its m, its sum and its unnormalised
// out.
//
// Products run on the matrix cores with tokens as the rows of the first operand: S^T = K Q^T leaves a lane with
// scores of one query row (its column) and the tokens of its own lane group, which is what the second product's
// operand P^T of O^T = V^T P^T holds: the weights never leave their lane.  A matrix product's inner index may be
// permuted, so K's values are read in 16-byte runs, and so are V's tokens taken in the order that S^T leaves.
#include "launch.h"
#include "paged.h"

#include <algorithm>

namespace {

using namespace kvsnap;

constexpr float kLog2e = 1.44269504088896340736f;

// ----------------------------------------------------------------- types and products

template <typename T>
struct Matrix;
template <>
struct Matrix<__bf16> {
    using Vec = bf16x8;
    static __device__ __forceinline__ f32x4 mul16(Vec a, Vec b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Matrix<_Float16> {
    using Vec = half8_t;
    static __device__ __forceinline__ f32x4 mul16(Vec a, Vec b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

// What the products run in: the cache's 16-bit type, or bf16 for an e4m3 cache, whose every value times its block's
// power of two is a bf16.  fp16 queries and weights are then two bf16 terms each, their first and the rest: 16 bits of
// the value, where one bf16 would lose three of fp16's.
template <typename Q, bool kEight>
struct Shape {
    using T = Q;
    static constexpr int kTerms = 1;
};
template <>
struct Shape<_Float16, true> {
    using T = __bf16;
    static constexpr int kTerms = 2;
};
template <>
struct Shape<__bf16, true> {
    using T = __bf16;
    static constexpr int kTerms = 1;
};

__device__ __forceinline__ void two_terms(float x, bf16x8& first, bf16x8& rest, int i) {
    first[i] = static_cast<__bf16>(x);
    rest[i] = static_cast<__bf16>(x - static_cast<float>(first[i]));
}

// kWords words from memory aligned to them (to 16 bytes, if they are more).
template <int kWords>
__device__ __forceinline__ void load_words(const char* from, uint32_t* to) {
    if constexpr (kWords == 1) {
        to[0] = *reinterpret_cast<const uint32_t*>(from);
    } else if constexpr (kWords == 2) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(from);
        to[0] = x[0], to[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
            const u32x4 x = reinterpret_cast<const u32x4*>(from)[i];
#pragma unroll
            for (int k = 0; k < 4; ++k) to[4 * i + k] = x[k];
        }
    }
}

__device__ __forceinline__ uint32_t two_bf16(uint32_t word, float scale, bool high) {
    return high ? bits<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, true))
                : bits<uint32_t>(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, false));
}

__device__ __forceinline__ float max_across_groups(float x) {
    // Lanes 16 and 32 apart hold the same row: the halves, then the quarters, change places.
    auto halves = __builtin_amdgcn_permlane32_swap(bits<uint32_t>(x), bits<uint32_t>(x), false, false);
    x = __builtin_fmaxf(bits<float>(halves[0]), bits<float>(halves[1]));
    auto quarters = __builtin_amdgcn_permlane16_swap(bits<uint32_t>(x), bits<uint32_t>(x), false, false);
    return __builtin_fmaxf(bits<float>(quarters[0]), bits<float>(quarters[1]));
}
__device__ __forceinline__ float sum_across_groups(float x) {
    auto halves = __builtin_amdgcn_permlane32_swap(bits<uint32_t>(x), bits<uint32_t>(x), false, false);
    x = bits<float>(halves[0]) + bits<float>(halves[1]);
    auto quarters = __builtin_amdgcn_permlane16_swap(bits<uint32_t>(x), bits<uint32_t>(x), false, false);
    return bits<float>(quarters[0]) + bits<float>(quarters[1]);
}

// ----------------------------------------------------------------- a row alone

struct Attend {
    kvsnap_paged_layer layer;
    kvsnap_sequences q;
    const void* query;
    void* out;
    float* lse;
    int64_t query_token_stride, query_head_stride, out_token_stride, out_head_stride;
    int tokens, heads, group;  // group: query heads that share a key head
    float scale;
    int window;                // 0: none
    int chunk, chunks;         // tokens a workgroup takes, and parts a row may have
    int head_tiles;            // of 16 heads, of a key head's
    Divider block_size;
    float* part;               // [tokens, heads, chunks, width] sums, then [tokens, heads, chunks, 2] largest and sum
};

constexpr int kTile = 32;         // tokens a wave takes at a time
constexpr int kWaves = 4;         // of a workgroup, side by side along the tokens
constexpr int kHeadTile = 16;     // query rows of a product

// What a row sees: tokens [low, high) of its sequence.
struct Sight {
    int sequence, low, high;
};

__device__ __forceinline__ Sight sight_of(const Attend& a, int row) {
    Sight sight{row, 0, 0};
    if (a.q.query_starts)
        sight.sequence = find_sequence(a.q.n_seqs, row, [&](int s) { return int64_t(a.q.query_starts[s]); });
    const Rows rows = rows_of(a.q, sight.sequence, a.tokens);
    const int i = row - rows.first;
    if (i < 0 || i >= rows.count) return Sight{-1, 0, 0};
    const int length = length_of(a.q, sight.sequence), position = length - rows.count + i;
    sight.low = a.window > 0 ? max(0, position + 1 - a.window) : 0;
    sight.high = min(position + 1, named_of(a.q, length, a.layer.block_size));
    return sight;
}

// Parts of a row's tokens, and the first token of part c: they start at the tile that holds the first seen token.
// The last part that there is room for takes what is left.
__device__ __forceinline__ int parts_of(const Attend& a, const Sight& sight) {
    const int first = sight.low & ~(kTile - 1);
    return sight.high <= sight.low ? 0 : min((sight.high - first + a.chunk - 1) / a.chunk, a.chunks);
}

// One wave's loads of a tile: K's rows for the first product and V's for the second.
template <bool kEight, int kJ>
struct Tile {
    static constexpr int kBytes = kEight ? 1 : 2;
    static constexpr int kRounds = kJ * kBytes / 4;         // 16-byte runs of a K row that a lane holds
    static constexpr int kWords = kJ * kBytes / 4;          // words of a V row that a lane holds
    u32x4 k[2][kRounds];
    uint32_t v[2][4][kWords];
    float k_scale[2], v_scale[2][4];                        // e4m3 only
};

// A row's heads of one key head over one part of its tokens, a workgroup of four waves that take tiles in turn.
//
// Bound by reading K and V once: 16 query rows of a product are used for `group` heads, a quarter of them for groups
// of four, and the matrix cores still wait for memory.
template <typename Q, bool kEight, int kJ, bool kWhole>
__global__ __launch_bounds__(kWaves * 64) void attend_row_kernel(Attend a) {
    using T = typename Shape<Q, kEight>::T;
    using Vec = typename Matrix<T>::Vec;
    constexpr int kTerms = Shape<Q, kEight>::kTerms;
    constexpr int kSteps = kJ / 2;                          // products of 32 values along a row
    using Loads = Tile<kEight, kJ>;
    constexpr int kRounds = Loads::kRounds, kWords = Loads::kWords, kBytes = Loads::kBytes;

    const int kv_heads = a.layer.kv_heads;
    uint32_t job = blockIdx.x;
    const int kv_head = job % kv_heads;
    job /= kv_heads;
    const int head_tile = job % a.head_tiles;
    job /= a.head_tiles;
    const int part = job % a.chunks;
    const int row = job / a.chunks;

    const Sight sight = sight_of(a, row);
    if (sight.sequence < 0) return;                         // padding
    const int parts = parts_of(a, sight);
    if (part >= max(parts, 1)) return;                      // the first part of a row that sees nothing writes zeros

    const int width = a.layer.width, size = a.layer.block_size;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int column = lane & 15, quarter = lane >> 4;
    const int first_head = kv_head * a.group + head_tile * kHeadTile;
    const int heads = min(kHeadTile, a.group - head_tile * kHeadTile);

    // Q^T: this lane's query head is its column.
    Vec q[kSteps][kTerms];
    {
        const Q* const from = static_cast<const Q*>(a.query) + row * a.query_token_stride +
                              (first_head + min(column, heads - 1)) * a.query_head_stride;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int at = kEight ? ((s >> 1) * 4 + quarter) * 16 + (s & 1) * 8 : s * 32 + quarter * 8;
            typename Matrix<Q>::Vec x{};
            if (at < width) x = *reinterpret_cast<const typename Matrix<Q>::Vec*>(from + at);
            if constexpr (kTerms == 1) {
                q[s][0] = x;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) two_terms(static_cast<float>(x[i]), q[s][0], q[s][1], i);
            }
        }
    }

    f32x4 sum[kJ];
#pragma unroll
    for (int j = 0; j < kJ; ++j) sum[j] = f32x4{0, 0, 0, 0};
    float top = -__builtin_inff(), total = 0;
    const float factor = a.scale * kLog2e;

    const int base = (sight.low & ~(kTile - 1)) + part * a.chunk;
    const int stop = part == a.chunks - 1 ? sight.high : min(sight.high, base + a.chunk);
    const int32_t* const table = a.q.block_tables + sight.sequence * a.q.table_stride;
    const char* const keys = static_cast<const char*>(a.layer.key) + kv_head * a.layer.head_stride * kBytes;
    const char* const values = static_cast<const char*>(a.layer.value) + kv_head * a.layer.head_stride * kBytes;
    const uint8_t* const scales = kEight ? a.layer.scales + kv_head * a.layer.scale_head_stride : nullptr;
    const int row_bytes = static_cast<int>(a.layer.token_stride) * kBytes;
    const int64_t block_bytes = a.layer.block_stride * kBytes;

    // Blocks of 16-token groups (kWhole: a block is whole groups): lane i holds that of group `cached` + i.
    int cached = -64, block_of = -1;
    float k_scale_of = 0, v_scale_of = 0;
    const auto block_at = [&](int token) -> int {           // of the table, -1 where there is none
        const uint32_t page = a.block_size.divide(token);
        if (page >= static_cast<uint32_t>(a.q.table_width) || token >= stop) return -1;
        const int block = table[page];
        return static_cast<uint32_t>(block) < static_cast<uint64_t>(a.layer.blocks) ? block : -1;
    };

    const auto load_k = [&](Loads& tile, int token) {
        if constexpr (kWhole) {
            const int group = token >> 4;
            if (group + 2 > cached + 64) {
                cached = group;
                block_of = block_at((group + lane) * 16);
                if constexpr (kEight) {
                    const uint8_t* const scale = scales + max(block_of, 0) * a.layer.scale_block_stride;
                    k_scale_of = power_of(scale[0]);
                    v_scale_of = power_of(scale[a.layer.scale_side_stride]);
                }
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int block, slot;
            if constexpr (kWhole) {
                const int at = token + 16 * h;
                block = __builtin_amdgcn_readlane(block_of, (at >> 4) - cached);
                slot = at - a.block_size.divide(at) * size + column;
                if constexpr (kEight)
                    tile.k_scale[h] = bits<float>(
                        __builtin_amdgcn_readlane(bits<int>(k_scale_of), (at >> 4) - cached));
            } else {
                const int at = token + 16 * h + column;
                block = block_at(at);
                slot = at - a.block_size.divide(at) * size;
                if constexpr (kEight)
                    tile.k_scale[h] = power_of(scales[max(block, 0) * a.layer.scale_block_stride]);
            }
            const char* const from = keys + block * block_bytes + slot * row_bytes;
#pragma unroll
            for (int r = 0; r < kRounds; ++r) {
                const int at = (r * 4 + quarter) * 16;      // bytes of the row
                tile.k[h][r] = u32x4{0, 0, 0, 0};
                if (block >= 0 && at < width * kBytes) tile.k[h][r] = *reinterpret_cast<const u32x4*>(from + at);
            }
        }
    };
    const auto load_v = [&](Loads& tile, int token) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                int block, slot;
                if constexpr (kWhole) {
                    const int at = token + 16 * h;
                    block = __builtin_amdgcn_readlane(block_of, (at >> 4) - cached);
                    slot = at - a.block_size.divide(at) * size + quarter * 4 + i;
                    if constexpr (kEight)
                        tile.v_scale[h][i] = bits<float>(
                            __builtin_amdgcn_readlane(bits<int>(v_scale_of), (at >> 4) - cached));
                } else {
                    const int at = token + 16 * h + quarter * 4 + i;
                    block = block_at(at);
                    slot = at - a.block_size.divide(at) * size;
                    if constexpr (kEight)
                        tile.v_scale[h][i] = power_of(
                            scales[max(block, 0) * a.layer.scale_block_stride + a.layer.scale_side_stride]);
                }
                const char* const from = values + block * block_bytes + slot * row_bytes + column * kJ * kBytes;
#pragma unroll
                for (int w = 0; w < kWords; ++w) tile.v[h][i][w] = 0;
                if (block >= 0 && column * kJ < width) load_words<kWords>(from, tile.v[h][i]);
            }
        }
    };

    const auto visible = [&](int token) { return token >= sight.low && token < stop; };
    // A token is seen if it is in sight and its block is one of the cache's.
    const auto seen_mask = [&](int token) -> uint32_t {     // bit 4h + i: token + 16 h + 4 quarter + i
        uint32_t mask = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = token + 16 * h + 4 * quarter + i;
                bool ok = visible(at);
                if constexpr (kWhole) ok = ok && __builtin_amdgcn_readlane(block_of, ((token >> 4) + h) - cached) >= 0;
                else ok = ok && block_at(at) >= 0;
                mask |= ok ? 1u << (4 * h + i) : 0;
            }
        return mask;
    };

    for (int token = base + wave * kTile; token < stop; token += kWaves * kTile) {
        Loads tile;
        load_k(tile, token);
        load_v(tile, token);
        const uint32_t mask = seen_mask(token);

        f32x4 score[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            score[h] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                Vec k;
                if constexpr (kEight) {
                    u32x4 two;
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        two[w] = two_bf16(tile.k[h][s >> 1][(s & 1) * 2 + (w >> 1)], tile.k_scale[h], w & 1);
                    k = bits<Vec>(two);
                } else {
                    k = bits<Vec>(tile.k[h][s]);
                }
#pragma unroll
                for (int t = 0; t < kTerms; ++t) score[h] = Matrix<T>::mul16(k, q[s][t], score[h]);
            }
        }

        float most = -__builtin_inff();
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                score[h][i] = mask >> (4 * h + i) & 1 ? score[h][i] : -__builtin_inff();
                most = __builtin_fmaxf(most, score[h][i]);
            }
        most = max_across_groups(most);
        if (__ballot(most > top)) {
            const float grown = __builtin_fmaxf(top, most);
            const float shrink = top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((top - grown) * factor);
            total *= shrink;
#pragma unroll
            for (int j = 0; j < kJ; ++j) sum[j] *= shrink;
            top = grown;
        }
        const float against = top == -__builtin_inff() ? 0.0f : top * factor;
        Vec p[kTerms];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(score[h][i], factor, -against));
                total += x;
                if constexpr (kTerms == 2) two_terms(x, p[0], p[1], 4 * h + i);
                else p[0][4 * h + i] = static_cast<T>(x);
            }

        // V^T: the tokens of this lane's column of values, from rows of values: pairs of 16-bit words change places.
        uint32_t wide[2][4][kJ / 2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool ok = mask >> (4 * h + i) & 1;    // what is not seen may hold anything: 0 * NaN is NaN
#pragma unroll
                for (int w = 0; w < kJ / 2; ++w) {
                    uint32_t word;
                    if constexpr (kEight) word = two_bf16(tile.v[h][i][w >> 1], tile.v_scale[h][i], w & 1);
                    else word = tile.v[h][i][w];
                    wide[h][i][w] = ok ? word : 0;
                }
            }
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
            u32x4 tokens;
#pragma unroll
            for (int w = 0; w < 4; ++w)
                tokens[w] = __builtin_amdgcn_perm(wide[w >> 1][(w & 1) * 2 + 1][j >> 1],
                                                  wide[w >> 1][(w & 1) * 2][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int t = 0; t < kTerms; ++t) sum[j] = Matrix<T>::mul16(bits<Vec>(tokens), p[t], sum[j]);
        }
    }

    // The waves' parts join in LDS: sums [wave][head][width], then the largest scores and totals.
    extern __shared__ float shared[];
    float* const tops = shared + kWaves * heads * width;
    float* const totals = tops + kWaves * kHeadTile;
    total = sum_across_groups(total);
    if (column < heads) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = (quarter * 4 + i) * kJ;
            if (at < width) {
#pragma unroll
                for (int j = 0; j < kJ; ++j) shared[(wave * heads + column) * width + at + j] = sum[j][i];
            }
        }
        if (quarter == 0) {
            tops[wave * kHeadTile + column] = top;
            totals[wave * kHeadTile + column] = total;
        }
    }
    __syncthreads();
    for (int at = threadIdx.x * 2; at < heads * width; at += kWaves * 64 * 2) {
        const int head = at / width, d = at - head * width;
        float most = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) most = __builtin_fmaxf(most, tops[w * kHeadTile + head]);
        float x = 0, y = 0, all = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float mine = tops[w * kHeadTile + head];
            const float share = mine == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((mine - most) * factor);
            const float* const from = shared + (w * heads + head) * width + d;
            x += from[0] * share;
            y += from[1] * share;
            all += totals[w * kHeadTile + head] * share;
        }
        const int64_t index = int64_t(row) * a.heads + first_head + head;
        if (parts > 1) {
            float* const to = a.part + (index * a.chunks + part) * width + d;
            to[0] = x;
            to[1] = y;
            if (d == 0) {
                float* const about = a.part + int64_t(a.tokens) * a.heads * a.chunks * width +
                                     (index * a.chunks + part) * 2;
                about[0] = most;
                about[1] = all;
            }
        } else {
            const float over = all > 0 ? 1.0f / all : all == 0 ? 0.0f : all;    // NaN stays
            Q* const to = static_cast<Q*>(a.out) + row * a.out_token_stride +
                          (first_head + head) * a.out_head_stride + d;
            to[0] = static_cast<Q>(x * over);
            to[1] = static_cast<Q>(y * over);
            if (a.lse && d == 0) a.lse[index] = most * a.scale + __builtin_logf(all);
        }
    }
}

// The parts of a row's head, joined: a workgroup's threads take values along the row and parts in turn.
template <typename Q>
__global__ __launch_bounds__(256) void join_kernel(Attend a) {
    const int head = blockIdx.x % a.heads, row = blockIdx.x / a.heads;
    const Sight sight = sight_of(a, row);
    if (sight.sequence < 0) return;
    const int parts = parts_of(a, sight);
    if (parts < 2) return;                                  // the row's own workgroup wrote it
    const int width = a.layer.width;
    const int64_t index = int64_t(row) * a.heads + head;
    const float* const from = a.part + index * a.chunks * width;
    const float* const about = a.part + int64_t(a.tokens) * a.heads * a.chunks * width + index * a.chunks * 2;
    const float factor = a.scale * kLog2e;
    float most = -__builtin_inff();
    for (int c = 0; c < parts; ++c) most = __builtin_fmaxf(most, about[2 * c]);
    for (int d = threadIdx.x; d < width; d += 256) {
        float x = 0, all = 0;
        for (int c = 0; c < parts; ++c) {
            const float mine = about[2 * c];
            const float share = mine == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((mine - most) * factor);
            x += from[c * width + d] * share;
            all += about[2 * c + 1] * share;
        }
        const float over = all > 0 ? 1.0f / all : all == 0 ? 0.0f : all;
        static_cast<Q*>(a.out)[row * a.out_token_stride + head * a.out_head_stride + d] = static_cast<Q>(x * over);
        if (a.lse && d == 0) a.lse[index] = most * a.scale + __builtin_logf(all);
    }
}

// ----------------------------------------------------------------- launches

// Tokens of a part, and parts of the longest row.
struct Split {
    int chunk, chunks;
};

Split split_of(int64_t jobs, int64_t longest) {
    constexpr int64_t least = 4 * kTile * kWaves, wanted = 2048;
    longest = std::max<int64_t>(longest, 1);
    int64_t chunk = std::max(least, longest * jobs / wanted);
    chunk = (chunk + kTile * kWaves - 1) / (kTile * kWaves) * (kTile * kWaves);
    return Split{static_cast<int>(std::min<int64_t>(chunk, 1 << 30)),
                 static_cast<int>((longest + kTile - 1 + chunk - 1) / chunk)};
}

// The tokens that a row may see, at most.
int64_t longest_sight(int64_t max_length, int64_t window) {
    return window > 0 ? std::min(window, max_length) : max_length;
}

template <typename Q, bool kEight, int kJ>
void launch_rows_of(const Attend& a, unsigned grid, unsigned lds, hipStream_t stream) {
    if (a.layer.block_size % 16 == 0)
        hipLaunchKernelGGL((attend_row_kernel<Q, kEight, kJ, true>), dim3(grid), dim3(kWaves * 64), lds, stream, a);
    else
        hipLaunchKernelGGL((attend_row_kernel<Q, kEight, kJ, false>), dim3(grid), dim3(kWaves * 64), lds, stream, a);
}

template <typename Q, bool kEight>
void launch_rows(const Attend& a, unsigned grid, unsigned lds, hipStream_t stream) {
    if (a.layer.width <= 64) launch_rows_of<Q, kEight, 4>(a, grid, lds, stream);
    else if (a.layer.width <= 128) launch_rows_of<Q, kEight, 8>(a, grid, lds, stream);
    else launch_rows_of<Q, kEight, 16>(a, grid, lds, stream);
}

template <typename Q>
void launch_attend(const Attend& a, hipStream_t stream) {
    const int64_t grid = int64_t(a.tokens) * a.chunks * a.head_tiles * a.layer.kv_heads;
    require(grid < (int64_t(1) << 31), "attend: too many rows for one launch");
    const unsigned lds = 4u * (kWaves * std::min(kHeadTile, a.group) * a.layer.width + 2 * kWaves * kHeadTile);
    if (a.layer.type == KVSNAP_E4M3) launch_rows<Q, true>(a, static_cast<unsigned>(grid), lds, stream);
    else launch_rows<Q, false>(a, static_cast<unsigned>(grid), lds, stream);
    check_launched("attend");
    if (a.chunks > 1) {
        hipLaunchKernelGGL(join_kernel<Q>, dim3(static_cast<unsigned>(a.tokens) * a.heads), dim3(256), 0, stream, a);
        check_launched("attend's join");
    }
}

}  // namespace

extern "C" {

size_t kvsnap_attend_workspace_bytes(int64_t tokens, int n_seqs, int heads, int kv_heads, int width,
                                     int64_t max_length, int64_t window) {
    (void)n_seqs;
    if (tokens <= 0 || heads <= 0 || kv_heads <= 0) return 0;
    const int64_t tiles = (heads / kv_heads + kHeadTile - 1) / kHeadTile;
    const Split split = split_of(tokens * kv_heads * tiles, longest_sight(max_length, window));
    return split.chunks < 2 ? 0 : static_cast<size_t>(tokens) * heads * split.chunks * (width + 2) * sizeof(float);
}

int kvsnap_attend(const kvsnap_paged_layer* layer, const kvsnap_sequences* sequences, const void* query,
                  int64_t query_token_stride, int64_t query_head_stride, void* out, int64_t out_token_stride,
                  int64_t out_head_stride, float* lse, int64_t tokens, int heads, int type, float scale,
                  int64_t window, int64_t max_length, void* workspace, size_t workspace_bytes, uintptr_t stream) {
    return guarded([&] {
        require(layer && sequences, "attend needs a layer and its sequences");
        check_layer(*layer);
        check_sequences(*sequences, *layer);
        require(tokens >= 0 && tokens < (int64_t(1) << 31) && heads >= 0, "attend: bad size");
        require(window >= 0 && max_length >= 0, "attend: negative window or length");
        require(scale > 0 && scale < 1e30f, "attend: the scale must be positive and finite");
        if (tokens == 0 || heads == 0 || sequences->n_seqs == 0) return;
        require(heads % layer->kv_heads == 0, "attend: query heads must be a multiple of the cache's");
        require(sequences->query_starts || tokens == sequences->n_seqs,
                "attend: without query_starts every sequence has one row");
        require(type == KVSNAP_BF16 || type == KVSNAP_FP16, "attend: queries must be bf16 or fp16");
        require(layer->type == KVSNAP_E4M3 || layer->type == type, "attend: a 16-bit cache must have the queries' type");
        require(query && out, "attend needs device pointers");
        require(reinterpret_cast<uintptr_t>(query) % 16 == 0 && query_token_stride * 2 % 16 == 0 &&
                    query_head_stride * 2 % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                    out_token_stride * 2 % 16 == 0 && out_head_stride * 2 % 16 == 0,
                "attend: rows and heads must be 16-byte aligned");
        Attend a{};
        a.layer = *layer;
        a.q = *sequences;
        a.query = query;
        a.out = out;
        a.lse = lse;
        a.query_token_stride = query_token_stride, a.query_head_stride = query_head_stride;
        a.out_token_stride = out_token_stride, a.out_head_stride = out_head_stride;
        a.tokens = static_cast<int>(tokens), a.heads = heads, a.group = heads / layer->kv_heads;
        a.scale = scale;
        a.window = static_cast<int>(std::min<int64_t>(window, (int64_t(1) << 31) - 1));
        a.head_tiles = (a.group + kHeadTile - 1) / kHeadTile;
        a.block_size = Divider::of(layer->block_size);
        const int64_t named = int64_t(sequences->table_width) * layer->block_size;
        const Split split = split_of(tokens * layer->kv_heads * a.head_tiles,
                                     longest_sight(std::min(max_length, named), window));
        a.chunk = split.chunk, a.chunks = split.chunks;
        a.part = static_cast<float*>(workspace);
        require(workspace_bytes >= kvsnap_attend_workspace_bytes(tokens, sequences->n_seqs, heads, layer->kv_heads,
                                                                 layer->width, std::min(max_length, named), window),
                "attend: the workspace is too small");
        require(a.chunks < 2 || (workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                "attend: the workspace must be 16-byte aligned device memory");
        const auto launch = type == KVSNAP_BF16 ? launch_attend<__bf16> : launch_attend<_Float16>;
        launch(a, reinterpret_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
