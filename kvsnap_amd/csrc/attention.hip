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
#include <type_traits>

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
    static __device__ __forceinline__ f32x16 mul32(Vec a, Vec b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Matrix<_Float16> {
    using Vec = half8_t;
    static __device__ __forceinline__ f32x4 mul16(Vec a, Vec b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mul32(Vec a, Vec b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

// What the products run in: the cache's 16-bit type, or bf16 for an e4m3 cache, whose every value times its block's
// power of two is a bf16 (from 2^-117 to 2^119; the bits of e4m3's least values fall out below, its largest are infinite
// above).  fp16 queries and weights are then two bf16 terms each, their first and the rest: 16 bits of
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

// What weights are relative to: a score near the largest so far, `slack` binary logarithms below it at most.
//
// Weights of an fp16 cache's values are fp16 too, whose range is short: below 2^-14 they lose bits, at 2^-25 they are
// gone from the product while they count in the sum.  So they are 2^kLift times as large, fp16's range from its top
// down, and their reference follows the tiles' largest scores down as well as up: where one is more than kFall under it,
// it moves to just below that.  A weight is then rounded by half a step, or by 2^-25 where its tile's largest is at least
// 2^(kLift - kFall): whatever the length, that moves a row's out by at most the tile's tokens (64, or 32 for rows alone)
// times 2^-30 of the largest value.
template <typename T>
struct Weights {
    static constexpr bool kFollow = std::is_same_v<T, _Float16>;
    static constexpr float kLift = kFollow ? 9 : 0, kDrop = kFollow ? 0x1p-9f : 1;      // kDrop: 2^-kLift
    static constexpr float kFall = 4;
    float factor, slack, fall;

    __device__ __forceinline__ Weights(float factor, float slack_of)
        : factor(factor), slack(slack_of > 0 ? __builtin_fminf(slack_of / factor, 1e30f) : 0),
          fall(__builtin_fminf(kFall / factor, 1e30f)) {}

    // Whether a row's reference moves for scores of at most `most`, and where to.  Down no farther than sums of `total`,
    // the row's, have room to grow: to 2^90, and values are at most 2^16.
    __device__ __forceinline__ bool moves(float top, float most) const {
        return most - top > slack || (kFollow && most - top < -fall);
    }
    __device__ __forceinline__ float moved(float top, float most, float total) const {
        if (!kFollow) return __builtin_fmaxf(top, most);
        if (most == -__builtin_inff() || !moves(top, most)) return top;
        const float below = most - __builtin_fminf(1.0f / factor, 1e30f);
        if (!(below < top)) return below;
        return __builtin_fmaxf(below, top - __builtin_fmaxf(90.0f - __builtin_log2f(total), 0.0f) / factor);
    }
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

__device__ __forceinline__ float max_across_halves(float x) {
    auto halves = __builtin_amdgcn_permlane32_swap(bits<uint32_t>(x), bits<uint32_t>(x), false, false);
    return __builtin_fmaxf(bits<float>(halves[0]), bits<float>(halves[1]));
}
__device__ __forceinline__ float sum_across_halves(float x) {
    auto halves = __builtin_amdgcn_permlane32_swap(bits<uint32_t>(x), bits<uint32_t>(x), false, false);
    return bits<float>(halves[0]) + bits<float>(halves[1]);
}

// Weights are 2^((score - top) * factor): the difference is exact for the tokens that count, however large the scores.
// Rows alone take it so.  Tiles, which are short of vector instructions, take 2^(score * factor - top * factor) by one
// operation a score: what rounding top * factor moves is common to a row's weights and falls out, while it is little.
// Whether some row's is more than 2^-14 (largest scores from some 2^10 binary logarithms on; from some 2^30 the powers
// overflow, or leave every weight 0) and tiles take the difference first too.
__device__ __forceinline__ bool rounds_far(float top, float factor) {
    return __ballot(!(__builtin_fabsf(__builtin_fmaf(top, factor, -(top * factor))) <= 0x1p-14f) &&
                    top != -__builtin_inff()) != 0;
}

// One over a row's sum: 0 for a row that sees nothing, and NaN stays.
__device__ __forceinline__ float over(float total) { return total > 0 ? 1.0f / total : total == 0 ? 0.0f : total; }

// ----------------------------------------------------------------- a row alone

// Tokens of a part, and parts that the longest row may have.
struct Split {
    int chunk, chunks;
};

// Where parts leave a head's unnormalised out, and its largest score and total.
struct Parts {
    float *sums, *totals;
};

// Rows alone, and tiles of rows: how their tokens are cut into workgroups' jobs.
struct RowJobs {
    int even;      // cut into equal parts, by the lengths that the sequences have, or `chunks` of `chunk` tiles each
    int chunk, chunks;
    int room, fitted;   // even: at least `chunk` tiles, for about `room` jobs, or no more than those
};

struct TileJobs {
    int even, room;     // cut into parts for up to `room` jobs more than there are tiles, or whole
};

// Sequences that a wave goes over, 64 at a time, to cut their rows' tokens evenly; more have parts of one length, by the
// longest.
constexpr int kEvenSeqs = 256;

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
    RowJobs rows;
    TileJobs tiles;
    Parts row_parts, tile_parts;  // [job, beside, heads of a tile], and [job, rows of a tile]
    int2* row_info;               // [sequence, heads' group]: the first job and the parts of rows alone
    int2* tile_info;              // [sequence, 2]: the first job of its tiles and their parts, tokens of a part and tiles
    int tile_jobs;                // that there is room for
    int least_rows;               // of a sequence whose rows are taken in tiles
    int head_tiles;            // of 16 heads, of a key head's
    int beside;                // key heads that a workgroup's waves take side by side
    int slots;                 // heads of a tile, at most
    Divider block_size, group_size, all_heads, quarter_width;
    uint32_t block_pieces, token_pieces;      // strides in 16 bytes
    uint32_t stage_pages, stage_slots;        // pages and slots that 64 tokens go on by
};

constexpr int kTile = 32;         // tokens a wave takes at a time
constexpr int kWaves = 8;         // of a workgroup
constexpr int kHeadTile = 16;     // query rows of a product

// What rows see, first to last: tokens [low, high) of their sequence, the first row at position `position`.
struct Sight {
    int low, high, position;
};

__device__ __forceinline__ Sight sight_of(const Attend& a, int sequence, const Rows& rows, int first, int last) {
    const int length = length_of(a.q, sequence), position = length - rows.count + first;
    return Sight{a.window > 0 ? max(0, position + 1 - a.window) : 0,
                 min(position + last - first + 1, named_of(a.q, length, a.layer.block_size)), position};
}

// Parts of what rows see: they start at the tile of tokens that holds the first seen token, and the last part that
// there is room for takes what is left.
template <int kTokens>
__device__ __forceinline__ int parts_of(const Split& split, const Sight& sight) {
    const int first = sight.low & ~(kTokens - 1);
    return sight.high <= sight.low ? 0 : min((sight.high - first + split.chunk - 1) / split.chunk, split.chunks);
}

// A job of the rows alone: a part of a sequence's tiles of tokens, for a workgroup's heads.
struct RowJob {
    int sequence, heads, part, parts, chunk;   // heads: which of the row's groups of heads; chunk: tiles of a part
    int64_t first;                             // the sequence's first job; its parts' lie `head_groups` apart
};

// Tiles of tokens that a sequence's one row sees; 1 where it sees nothing, which is written too, and 0 for a sequence
// of no or of more rows.
__device__ __forceinline__ int row_tiles(const Attend& a, int sequence) {
    const Rows rows = rows_of(a.q, sequence, a.tokens);
    if (rows.count != 1) return 0;
    const Sight sight = sight_of(a, sequence, rows, 0, 0);
    return max((sight.high - (sight.low & ~(kTile - 1)) + kTile - 1) / kTile, 1);
}

// Sums of the wave's values up to each lane's, by moves between lanes that need no LDS.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);     // from 1, 2, 4 and 8 lanes below, of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);     // lane 15 of 16 to the next 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);     // lane 31 to the upper half
    return x;
}
__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

__device__ __forceinline__ int64_t wave_sum64(int64_t x) {     // of values from 0 to 2^40
    return (int64_t(wave_sum(static_cast<int>(x >> 16))) << 16) + wave_sum(static_cast<int>(x & 0xffff));
}

// The sequence whose jobs hold `job`: its first job, its parts, and how long one is.
struct Cut {
    int sequence, parts, chunk;
    int64_t first;
};

// Work cut evenly over `room` jobs.  A lane holds the `units` of every 64th sequence (0: none of these jobs), `times`
// times over; a sequence has `each` jobs for every part and time.  Parts are whole multiples of `step` units, `least` at
// the least: `all` over `room`, or up to most_eighths / 8 of that, the shortest tried with which the jobs come out as no
// more than `room`.
template <int kTurns>
__device__ __forceinline__ Cut even_cut(int n_seqs, int64_t job, const int (&units)[kTurns], const int (&times)[kTurns],
                                        int each, int least, int step, int room, int most_eighths) {
    int64_t mine_of_all = 0;
#pragma unroll
    for (int i = 0; i < kTurns; ++i) mine_of_all += int64_t(units[i]) * times[i];
    const int64_t all = wave_sum64(mine_of_all);
    int chunk = 0;
#pragma unroll 1
    for (int eighths = 8; eighths <= most_eighths; ++eighths) {
        const int64_t share = (all * each * eighths + 8 * room - 1) / (8 * room);
        // (2^24 units are more than a sequence has, and their tokens still fit 32 bits)
        chunk = (static_cast<int>(min(max(int64_t(least), share), int64_t(1) << 24)) + step - 1) / step * step;
        if (eighths == most_eighths) break;
        int jobs = 0;
#pragma unroll
        for (int i = 0; i < kTurns; ++i) jobs += (units[i] + chunk - 1) / chunk * times[i];
        if (int64_t(wave_sum(jobs)) * each <= room) break;
    }
    int64_t before = 0;
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
        if (64 * i >= n_seqs) break;
        const int parts = (units[i] + chunk - 1) / chunk, mine = parts * times[i], up_to = wave_scan(mine);
        const uint64_t holds = __ballot(before + int64_t(up_to) * each > job);
        if (holds) {
            const int at = __builtin_ctzll(holds);
            const int upto_before = __builtin_amdgcn_readlane(up_to, at) - __builtin_amdgcn_readlane(mine, at);
            return Cut{64 * i + at, __builtin_amdgcn_readlane(parts, at), chunk, before + int64_t(upto_before) * each};
        }
        before += int64_t(__builtin_amdgcn_readlane(up_to, 63)) * each;
    }
    return Cut{-1, 0, 1, 0};
}

// The sequence whose jobs hold `job`, and its parts.
__device__ __forceinline__ RowJob row_job(const Attend& a, int64_t job, int head_groups) {
    if (!a.rows.even) {
        const int sequence = static_cast<int>(job / (a.rows.chunks * head_groups));
        const int64_t first = int64_t(sequence) * a.rows.chunks * head_groups;
        const int rest = static_cast<int>(job - first), tiles = row_tiles(a, sequence);
        // The last part that there is room for takes what is left.
        return RowJob{tiles ? sequence : -1, rest % head_groups, rest / head_groups,
                      min((tiles + a.rows.chunk - 1) / a.rows.chunk, a.rows.chunks), a.rows.chunk, first};
    }
    const int lane = __lane_id();
    int tiles[kEvenSeqs / 64], once[kEvenSeqs / 64];
#pragma unroll
    for (int i = 0; i < kEvenSeqs / 64; ++i) {      // what is past 2^29 tokens goes to a row's last part
        tiles[i] = 64 * i + lane < a.q.n_seqs ? min(row_tiles(a, 64 * i + lane), 1 << 24) : 0;
        once[i] = 1;
    }
    // In whole turns of a workgroup's waves.
    const Cut cut = even_cut(a.q.n_seqs, job, tiles, once, head_groups, a.rows.chunk, kWaves / a.beside, a.rows.room,
                             a.rows.fitted ? 12 : 8);
    const int rest = static_cast<int>(job - cut.first);
    return RowJob{cut.sequence, rest % head_groups, rest / head_groups, cut.parts, cut.chunk, cut.first};
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

// Waves of a SIMD that attend_row_kernel's registers leave room for.  Two terms over blocks that are no whole groups of
// 16 tokens spill at four, and take 7 % longer than at two.
template <typename Q, bool kEight, int kJ, bool kWhole>
constexpr int row_waves() {
    return kEight && kJ <= 8 && (kWhole || Shape<Q, kEight>::kTerms == 1) ? 4 : 2;
}

// A row's heads of `beside` key heads over one part of its tokens, a workgroup of eight waves; those of one key head take
// its tiles of 32 tokens in turn.
//
// Bound by reading K and V once: 16 query rows of a product are used for `group` heads, a quarter of them for groups
// of four, and the matrix cores still wait for memory.  Loads go straight to the registers that the products take, as no
// wave shares them; sixteen waves a CU are what hides their latency (a tile's loads ahead of their use, at eight waves,
// measured the same).  64 ragged rows over 322 MB of e4m3 take 68 us (a kernel trace's), 4.8 TB/s where a plain read of
// as much reaches 6.6, and 7 for the join; what is missing is the start, four loads that follow from one another (length,
// table, rows), and the last workgroups' end.  Loads that keep out of the caches (nontemporal) are 5 % faster there and
// up to 45 % slower where a cache fits what the chip's does.
template <typename Q, bool kEight, int kJ, bool kWhole, bool kExact>
__global__ __launch_bounds__(kWaves * 64, (row_waves<Q, kEight, kJ, kWhole>())) void attend_row_kernel(Attend a) {
    using T = typename Shape<Q, kEight>::T;
    using Vec = typename Matrix<T>::Vec;
    using W = Weights<T>;
    constexpr int kTerms = Shape<Q, kEight>::kTerms;
    constexpr int kSteps = kJ / 2;                          // products of 32 values along a row
    using Loads = Tile<kEight, kJ>;
    constexpr int kRounds = Loads::kRounds, kWords = Loads::kWords, kBytes = Loads::kBytes;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int column = lane & 15, quarter = lane >> 4;
    // `beside` waves take key heads side by side, and those of one key head its tiles in turn.
    const int beside = a.beside, in_turn = kWaves / beside, turn = wave / beside;
    const int head_groups = a.layer.kv_heads / beside * a.head_tiles;
    const RowJob job = row_job(a, blockIdx.x, head_groups);
    if (job.sequence < 0 || job.part >= job.parts) return;
    const int sequence = job.sequence, part = job.part, parts = job.parts;
    if (a.row_info && part == 0 && threadIdx.x == 0)
        a.row_info[int64_t(sequence) * head_groups + job.heads] = int2{static_cast<int>(job.first), parts};
    const int kv_head = job.heads / a.head_tiles * beside + wave % beside, head_tile = job.heads % a.head_tiles;
    const Rows rows = rows_of(a.q, sequence, a.tokens);
    const int row = rows.first;
    const Sight sight = sight_of(a, sequence, rows, 0, 0);

    const int width = a.layer.width, size = a.layer.block_size;
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
    const W weights(factor, W::kFollow ? 6 : 0);

    const int base = (sight.low & ~(kTile - 1)) + part * job.chunk * kTile;
    const int stop = part == parts - 1 ? sight.high : min(sight.high, base + job.chunk * kTile);
    const int32_t* const table = a.q.block_tables + sequence * a.q.table_stride;
    const char* const keys = static_cast<const char*>(a.layer.key) + kv_head * a.layer.head_stride * kBytes;
    const char* const values = static_cast<const char*>(a.layer.value) + kv_head * a.layer.head_stride * kBytes;
    const uint8_t* const scales = kEight ? a.layer.scales + kv_head * a.layer.scale_head_stride : nullptr;
    const int row_bytes = static_cast<int>(a.layer.token_stride) * kBytes;
    const int64_t block_bytes = a.layer.block_stride * kBytes;

    const auto block_at = [&](int token) -> int {           // of the table, -1 where there is none
        const uint32_t page = a.block_size.divide(token);
        if (page >= static_cast<uint32_t>(a.q.table_width) || token >= stop) return -1;
        const int block = table[page];
        return static_cast<uint32_t>(block) < static_cast<uint64_t>(a.layer.blocks) ? block : -1;
    };
    // kWhole: lane i holds the block of the 16-token group `cached` + i, and its scales.
    int cached = -64, block_of = -1;
    float k_scale_of = 0, v_scale_of = 0;
    const uint32_t k_lane = column * row_bytes + quarter * 16;
    uint32_t v_lane[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v_lane[i] = (quarter * 4 + i) * row_bytes + (column * kJ < width ? column * kJ * kBytes : 0);

    // A tile's rows: 16 tokens by 16 lanes for K, four by a lane for V.  A block that the table does not name is read as
    // block 0, and its tokens are masked.
    Loads tile;
    uint32_t mask = 0;          // bit 4 h + i: this lane's token 16 h + 4 quarter + i is seen
    int64_t whole_offset[2];    // kWhole: where the tile's two groups of 16 tokens are
    const auto load_k = [&](int token) {
        mask = 0xff;
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
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = token + 16 * h;
                const int block = __builtin_amdgcn_readlane(block_of, (at >> 4) - cached);
                whole_offset[h] = max(block, 0) * block_bytes +
                                  int64_t(at - a.block_size.divide(at) * size) * row_bytes;
                if (block < 0) mask &= ~(0xfu << (4 * h));
#pragma unroll
                for (int r = 0; r < kRounds; ++r) {
                    if (kExact || r * 64 + quarter * 16 < width * kBytes)
                        tile.k[h][r] = *reinterpret_cast<const u32x4*>(keys + whole_offset[h] + k_lane + r * 64);
                    else
                        tile.k[h][r] = u32x4{0, 0, 0, 0};
                }
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = token + 16 * h + column;
                const int block = max(block_at(at), 0), slot = at - a.block_size.divide(at) * size;
                const int64_t offset = block * block_bytes + int64_t(slot) * row_bytes;
#pragma unroll
                for (int r = 0; r < kRounds; ++r) {
                    tile.k[h][r] = u32x4{0, 0, 0, 0};
                    if (r * 64 + quarter * 16 < width * kBytes)
                        tile.k[h][r] = *reinterpret_cast<const u32x4*>(keys + offset + r * 64 + quarter * 16);
                }
                if constexpr (kEight) tile.k_scale[h] = power_of(scales[block * a.layer.scale_block_stride]);
            }
        }
        if (token < sight.low || token + kTile > stop) {
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const int at = token + 16 * (t >> 2) + 4 * quarter + (t & 3);
                if (at < sight.low || at >= stop) mask &= ~(1u << t);
            }
        }
    };
    const auto load_v = [&](int token) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (kWhole) {
                    load_words<kWords>(values + whole_offset[h] + v_lane[i], tile.v[h][i]);
                } else {
                    const int at = token + 16 * h + quarter * 4 + i;
                    const int named = block_at(at), block = max(named, 0);
                    if (named < 0) mask &= ~(1u << (4 * h + i));
                    const int64_t offset = block * block_bytes + int64_t(at - a.block_size.divide(at) * size) * row_bytes;
                    load_words<kWords>(values + offset + v_lane[i] - (quarter * 4 + i) * row_bytes, tile.v[h][i]);
                    if constexpr (kEight)
                        tile.v_scale[h][i] =
                            power_of(scales[block * a.layer.scale_block_stride + a.layer.scale_side_stride]);
                }
            }
        if constexpr (kWhole && kEight) {       // behind the loads, which do not wait for them
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = (token >> 4) + h - cached;
                tile.k_scale[h] = bits<float>(__builtin_amdgcn_readlane(bits<int>(k_scale_of), at));
                tile.v_scale[h][0] = bits<float>(__builtin_amdgcn_readlane(bits<int>(v_scale_of), at));
            }
        }
    };

    for (int token = base + turn * kTile; token < stop; token += in_turn * kTile) {
        load_k(token);
        load_v(token);
        const uint32_t seen = mask;
        const bool ragged = __ballot(seen != 0xff) != 0;    // in most tiles every token is seen by every row

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
        if (ragged) {
#pragma unroll
            for (int t = 0; t < 8; ++t)
                score[t >> 2][t & 3] = seen >> t & 1 ? score[t >> 2][t & 3] : -__builtin_inff();
        }
        float most = -__builtin_inff();
#pragma unroll
        for (int t = 0; t < 8; ++t) most = __builtin_fmaxf(most, score[t >> 2][t & 3]);
        most = max_across_groups(most);
        if (__ballot(weights.moves(top, most))) {
            const float to = weights.moved(top, most, W::kFollow ? sum_across_groups(total) : 0);
            const float shrink = top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((top - to) * factor);
            total *= shrink;
#pragma unroll
            for (int j = 0; j < kJ; ++j) sum[j] *= shrink;
            top = to;
        }
        const float from = top == -__builtin_inff() ? 0.0f : top;
        Vec p[kTerms];
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(score[t >> 2][t & 3] - from, factor, W::kLift));
            total += x;
            if constexpr (kTerms == 2) two_terms(x, p[0], p[1], t);
            else p[0][t] = static_cast<T>(x);
        }

        // V^T: the tokens of this lane's column of values, from rows of values: pairs of 16-bit words change places.
        uint32_t wide[2][4][kJ / 2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int w = 0; w < kJ / 2; ++w) {
                    if constexpr (kEight)
                        wide[h][i][w] = two_bf16(tile.v[h][i][w >> 1], tile.v_scale[h][kWhole ? 0 : i], w & 1);
                    else
                        wide[h][i][w] = tile.v[h][i][w];
                }
        if (ragged) {       // what is not seen may hold anything: 0 * NaN is NaN
#pragma unroll
            for (int t = 0; t < 8; ++t)
#pragma unroll
                for (int w = 0; w < kJ / 2; ++w)
                    wide[t >> 2][t & 3][w] = seen >> t & 1 ? wide[t >> 2][t & 3][w] : 0;
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

    // The waves of a key head join in LDS: sums [wave][head][width], then the largest scores and totals.
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
    for (int at = (turn * 64 + lane) * 2; at < heads * width; at += in_turn * 64 * 2) {
        const int head = at / width, d = at - head * width;
        float most = -__builtin_inff();
        for (int w = wave % beside; w < kWaves; w += beside)
            most = __builtin_fmaxf(most, tops[w * kHeadTile + head]);
        float x = 0, y = 0, all = 0;
        for (int w = wave % beside; w < kWaves; w += beside) {
            const float mine = tops[w * kHeadTile + head];
            const float share = mine == -__builtin_inff() ? 0.0f
                                                           : __builtin_amdgcn_exp2f((mine - most) * factor) * W::kDrop;
            const float* const from = shared + (w * heads + head) * width + d;
            x += from[0] * share;
            y += from[1] * share;
            all += totals[w * kHeadTile + head] * share;
        }
        if (parts > 1) {
            const int64_t at_part = (int64_t(blockIdx.x) * beside + wave % beside) * a.slots + head;
            *reinterpret_cast<float2*>(a.row_parts.sums + at_part * width + d) = float2{x, y};
            if (d == 0) *reinterpret_cast<float2*>(a.row_parts.totals + at_part * 2) = float2{most, all};
        } else {
            typedef Q Two __attribute__((ext_vector_type(2)));
            const float share = over(all);
            *reinterpret_cast<Two*>(static_cast<Q*>(a.out) + row * a.out_token_stride +
                                    (first_head + head) * a.out_head_stride + d) =
                Two{static_cast<Q>(x * share), static_cast<Q>(y * share)};
            if (a.lse && d == 0)
                a.lse[int64_t(row) * a.heads + first_head + head] = most * a.scale + __builtin_logf(all);
        }
    }
}

// ----------------------------------------------------------------- rows in tiles

constexpr int kTileRows = 128;    // rows of a workgroup: (token, head) pairs that share a key head, heads fastest
constexpr int kTileWaves = 4;     // 32 rows each, the columns of a product
constexpr int kTileTokens = 64;   // tokens staged at a time
constexpr int kTileSeqs = 512;    // sequences at most where tiles are cut
constexpr int kLeastStages = 8;   // of 64 tokens, of a part

// The tile of a sequence's rows that starts at pair `first`: the tokens of its first and last pair.
__device__ __forceinline__ Sight tile_sight(const Attend& a, int sequence, const Rows& rows, int first) {
    const int last = min(first + kTileRows, rows.count * a.group) - 1;
    return sight_of(a, sequence, rows, a.group_size.divide(first), a.group_size.divide(last));
}

// A workgroup's job: a part of what a tile of a sequence's rows sees, for a key head.
struct TileJob {
    int sequence, kv_head, part;
    int64_t pair;       // the tile's first
    Split split;
};

// Tiles whole.  Sequence s has slots from query_starts[s] * group / 128 + s on: n rows have at most n * group / 128 + 1
// tiles.  Later ones see more tokens: they go first.
__device__ __forceinline__ TileJob whole_tile_job(const Attend& a, uint32_t job, uint32_t jobs) {
    const auto slots = [&](int s) {
        return int64_t(min(max(a.q.query_starts[s], 0), a.tokens)) * a.group / kTileRows + s;
    };
    const int64_t slot = (jobs - 1 - job) / a.layer.kv_heads;
    const int sequence = find_sequence(a.q.n_seqs, slot, slots);
    return TileJob{sequence, static_cast<int>(job % a.layer.kv_heads), 0, (slot - slots(sequence)) * kTileRows,
                   Split{1 << 29, 1}};
}

// Tiles in parts, by the lengths that the sequences have: a sequence's tiles are cut as its last is.  The workgroups of
// one key head's tiles follow one another by the number of key heads.
__device__ __forceinline__ TileJob even_tile_job(const Attend& a, uint32_t job) {
    constexpr int kTurns = kTileSeqs / 64;
    const int lane = __lane_id(), kv_heads = a.layer.kv_heads;
    int stages[kTurns], tiles[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
        const int s = 64 * i + lane;
        stages[i] = tiles[i] = 0;
        if (s >= a.q.n_seqs) continue;
        const Rows rows = rows_of(a.q, s, a.tokens);
        if (rows.count < a.least_rows) continue;
        tiles[i] = (rows.count * a.group + kTileRows - 1) / kTileRows;
        const Sight sight = tile_sight(a, s, rows, (tiles[i] - 1) * kTileRows);
        stages[i] = min(max((sight.high - (sight.low & ~(kTileTokens - 1)) + kTileTokens - 1) / kTileTokens, 1), 1 << 23);
    }
    const Cut cut = even_cut(a.q.n_seqs, job, stages, tiles, kv_heads, kLeastStages, 1, a.tiles.room, 12);
    if (cut.sequence < 0) return TileJob{-1, 0, 0, 0, Split{1, 1}};
    int tiles_of = 0;
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
        if (cut.sequence >> 6 == i) tiles_of = __builtin_amdgcn_readlane(tiles[i], cut.sequence & 63);
    const int rest = static_cast<int>(job - cut.first), time = rest / kv_heads;
    const Split split{cut.chunk * kTileTokens, cut.parts};
    if (rest == 0 && threadIdx.x == 0) {
        a.tile_info[2 * cut.sequence] = int2{static_cast<int>(cut.first), cut.parts};
        a.tile_info[2 * cut.sequence + 1] = int2{split.chunk, tiles_of};
    }
    return TileJob{cut.sequence, rest % kv_heads, time / tiles_of, int64_t(time % tiles_of) * kTileRows, split};
}

// Whether a pair of 16-bit values holds one that is not finite (`ones`: the type's exponent bits, twice).
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t word) {
    constexpr uint32_t ones = sizeof(T) == 2 && __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
    return ((word & ones) == ones ? 0xffffu : 0u) | ((word >> 16 & ones) == ones ? 0xffff0000u : 0u);
}

// A prompt's rows: 128 of them by 64 tokens at a time, K and V staged in LDS in the products' type, two buffers deep:
// the next tokens' loads are under way while the present ones' products run, and one barrier parts the two.
//
// K's rows are 16 bytes longer than the values (an odd number of 16-byte pieces: 16-byte reads down a column of rows
// meet every bank); V's are 64 or 192 bytes past a multiple of 256, so that the 64 bytes of four rows that half a wave's
// transposing read takes lie side by side over the banks.  No read waits for a bank.
//
// An 8k prompt of 32 heads over 8 of 128 in bf16 takes 633 us, 868 TFLOP/s of the products that its mask leaves, where a
// large plain product reaches 1280 on this card.  A stage costs a wave 1024 cycles of products and about 1100 of vector
// instructions (32 scores a lane: a multiplication, an exponential, a sum, half a rounding, half a maximum), and the two
// waves of a SIMD overlap little of the two.  Tried and slower: the next stage's scores between this stage's
// exponentials (1.6 times as long at 256 registers, and 1.2 times at width 64, where nothing spills), and higher priority
// for waves in their products (3 % longer).  Widths above 128 take the registers and LDS of a whole CU: one workgroup each.
template <typename Q, bool kEight, int kD, bool kWhole>
__global__ __launch_bounds__(kTileWaves * 64, kD <= 128 ? 2 : 1) void attend_tile_kernel(Attend a) {
    using T = typename Shape<Q, kEight>::T;
    using Vec = typename Matrix<T>::Vec;
    using W = Weights<T>;
    constexpr int kTerms = Shape<Q, kEight>::kTerms;
    constexpr int kBytes = kEight ? 1 : 2;
    constexpr int kSteps = kD / 16, kBlocks = kD / 32;
    constexpr int kPieces = kD / 8;                         // of eight values, of a row
    // Threads side by side along a row, so that a wave's rows lie in one group of 16 tokens.
    constexpr int kBeside = kPieces <= 8 ? 8 : kPieces <= 16 ? 16 : 32;
    constexpr int kLoads = kTileTokens * kBeside / (kTileWaves * 64);
    constexpr int kKeyRow = kD * 2 + 16, kValueRow = kD * 2 + (kD == 96 ? 0 : 64);
    constexpr int kStage = kTileTokens * (kKeyRow + kValueRow);
    constexpr uint32_t kNowhere = ~0u;
    __shared__ __attribute__((aligned(16))) char stage[2 * kStage];
    __shared__ uint32_t odd[3][2];                          // tokens with a value that is not finite, by turns

    const TileJob job = a.tiles.even ? even_tile_job(a, blockIdx.x) : whole_tile_job(a, blockIdx.x, gridDim.x);
    if (job.sequence < 0) return;
    const auto same = [](int x) { return __builtin_amdgcn_readfirstlane(x); };      // kept in scalar registers
    const int sequence = same(job.sequence), kv_head = same(job.kv_head), part = same(job.part);
    const Rows rows = rows_of(a.q, sequence, a.tokens);
    const int pairs = rows.count * a.group;
    if (rows.count < a.least_rows || job.pair < 0 || job.pair >= pairs) return;     // no rows, or a row alone
    const int pair0 = same(static_cast<int>(job.pair));
    const Split split{same(job.split.chunk), same(job.split.chunks)};
    const Sight sight = tile_sight(a, sequence, rows, pair0);
    const int parts = parts_of<kTileTokens>(split, sight);
    if (part >= max(parts, 1)) return;

    const int width = a.layer.width;
    const int thread = threadIdx.x, lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const int column = lane & 31, half = lane >> 5;

    // This lane's row, and the positions of the wave's first and last.
    const int pair = pair0 + wave * 32 + column;
    const bool real = pair < pairs;
    const int token_of = a.group_size.divide(min(pair, pairs - 1)), head_of = min(pair, pairs - 1) - token_of * a.group;
    const int place0 = length_of(a.q, sequence) - rows.count;
    const int position = place0 + token_of;
    const int wave_first = pair0 + wave * 32;
    const bool idle = wave_first >= pairs;
    const int low_position = place0 + static_cast<int>(a.group_size.divide(min(wave_first, pairs - 1)));
    const int high_position = place0 + static_cast<int>(a.group_size.divide(min(wave_first + 31, pairs - 1)));
    const int after = a.window > 0 ? position - a.window : -1;      // the row sees tokens behind this one, up to its own
    const int64_t row = rows.first + token_of;
    const int head = kv_head * a.group + head_of;

    Vec q[kSteps][kTerms];
    {
        const Q* const from = static_cast<const Q*>(a.query) + row * a.query_token_stride + head * a.query_head_stride;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int at = s * 16 + half * 8;
            typename Matrix<Q>::Vec x{};
            if (real && at < width) x = *reinterpret_cast<const typename Matrix<Q>::Vec*>(from + at);
            if constexpr (kTerms == 1) {
                q[s][0] = x;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) two_terms(static_cast<float>(x[i]), q[s][0], q[s][1], i);
            }
        }
    }

    const int base = (sight.low & ~(kTileTokens - 1)) + part * split.chunk;
    const int stop = part == split.chunks - 1 ? sight.high : min(sight.high, base + split.chunk);
    const int32_t* const table = a.q.block_tables + sequence * a.q.table_stride;
    const char* const keys = static_cast<const char*>(a.layer.key) + kv_head * a.layer.head_stride * kBytes;
    const char* const values = static_cast<const char*>(a.layer.value) + kv_head * a.layer.head_stride * kBytes;
    const uint8_t* const scales = kEight ? a.layer.scales + kv_head * a.layer.scale_head_stride : nullptr;

    // Where 64 tokens' rows are: lane i has token i's, or (kWhole: a block is whole groups of 16 tokens) those of group
    // i & 3.  The table is read two stages ahead of its use, a stage ahead of the rows, so that no wait for it is a wait
    // for them; pages and slots go on from stage to stage.
    struct Places {
        uint32_t at;                                        // in 16 bytes; kNowhere: in no block, or out of the part
        uint32_t k_scale, v_scale;                          // e8m0 bytes
    };
    const int lane_token = kWhole ? (lane & 3) * 16 : lane;
    uint32_t page = a.block_size.divide(base + lane_token), slot = base + lane_token - page * a.block_size.d;
    const auto named_block = [&](int token) {               // the table's entry for `page`; -1 where there is none
        int block = -1;
        if (token + lane_token + (kWhole ? 15 : 0) >= sight.low && token + lane_token < stop &&
            page < static_cast<uint32_t>(a.q.table_width))
            block = table[page];
        return block;
    };
    const auto places_of = [&](int block) {
        Places places{kNowhere, 127, 127};
        const bool named = static_cast<uint32_t>(block) < static_cast<uint32_t>(a.layer.blocks);
        if (named) places.at = static_cast<uint32_t>(block) * a.block_pieces + slot * a.token_pieces;
        if constexpr (kEight)
            if (named) {
                const uint8_t* const scale = scales + block * a.layer.scale_block_stride;
                places.k_scale = scale[0];
                places.v_scale = scale[a.layer.scale_side_stride];
            }
        page += a.stage_pages;
        slot += a.stage_slots;
        if (slot >= a.block_size.d) slot -= a.block_size.d, ++page;
        return places;
    };
    // Which of the 64 tokens are there.
    const auto valid_of = [&](const Places& places, int token) -> uint64_t {
        uint64_t valid = __ballot(places.at != kNowhere);
        if constexpr (kWhole) {
            const uint64_t groups = valid & 15;
            if (groups == 15 && token >= sight.low && token + kTileTokens <= stop) return ~uint64_t(0);
            valid = ((groups & 1) | (groups & 2) << 15 | (groups & 4) << 30 | (groups & 8) << 45) * 0xffff;
            if (token < sight.low) valid &= ~uint64_t(0) << min(sight.low - token, 63);
            if (token + kTileTokens > stop) valid &= ~uint64_t(0) >> min(kTileTokens - (stop - token), 63);
        }
        return valid;
    };
    // A thread's pieces of a stage.
    //
    // Threads past a narrower head's width load its first piece again and store it where that goes: no branch parts the
    // loads (one took an 8k prompt 24 % longer).  K's columns past the width stay 0, for the queries' zeros there to meet.
    const int my_row = thread / kBeside, my_place = thread - my_row * kBeside;
    const int my_piece = my_place * 8 < width ? my_place : 0;
    const uint32_t my_offset = (my_row & 15) * a.token_pieces * 16 + my_piece * 8 * kBytes;
    uint32_t k_words[kLoads][kEight ? 2 : 4] = {}, v_words[kLoads][kEight ? 2 : 4] = {};
    const auto load = [&](const Places& places, uint64_t valid) {
        if (kWhole && valid == ~uint64_t(0)) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                // The wave's group of 16 tokens, and where in it the pass begins.
                const int first_row = i * (kTileWaves * 64 / kBeside);
                const int group = (first_row + wave * (64 / kBeside)) >> 4;
                // (32 unsigned bits: the builtin's int would take a place from 32 GiB on as one below the cache)
                const uint32_t place = __builtin_amdgcn_readlane(places.at, group);
                const int64_t at = (int64_t(place) << 4) + (first_row & 15) * int64_t(a.token_pieces) * 16;
                load_words<kEight ? 2 : 4>(keys + at + my_offset, k_words[i]);
                load_words<kEight ? 2 : 4>(values + at + my_offset, v_words[i]);
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int row_of = i * (kTileWaves * 64 / kBeside) + my_row;
            const uint32_t at = __shfl(places.at, kWhole ? row_of >> 4 : row_of);
#pragma unroll
            for (int w = 0; w < (kEight ? 2 : 4); ++w) k_words[i][w] = v_words[i][w] = 0;
            if (valid >> row_of & 1) {
                const int64_t offset = (int64_t(at + (kWhole ? (row_of & 15) * a.token_pieces : 0)) << 4) +
                                       my_piece * 8 * kBytes;
                load_words<kEight ? 2 : 4>(keys + offset, k_words[i]);
                load_words<kEight ? 2 : 4>(values + offset, v_words[i]);
            }
        }
    };
    const auto store = [&](const Places& places, char* to, bool ragged, uint32_t* odd_tokens) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int row_of = i * (kTileWaves * 64 / kBeside) + my_row;
            u32x4 k, v;
            if constexpr (kEight) {
                const int from = (i * (kTileWaves * 64 / kBeside) + wave * (64 / kBeside)) >> 4;
                const float k_scale = power_of(kWhole ? __builtin_amdgcn_readlane(places.k_scale, from)
                                                      : __shfl(places.k_scale, row_of));
                const float v_scale = power_of(kWhole ? __builtin_amdgcn_readlane(places.v_scale, from)
                                                      : __shfl(places.v_scale, row_of));
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    k[w] = two_bf16(k_words[i][w >> 1], k_scale, w & 1);
                    v[w] = two_bf16(v_words[i][w >> 1], v_scale, w & 1);
                }
            } else {
#pragma unroll
                for (int w = 0; w < 4; ++w) k[w] = k_words[i][w], v[w] = v_words[i][w];
            }
            if (ragged) {
                // Some rows do not see some of these tokens, and a weight of 0 does not hide NaN: such values stay
                // out of the product and are added apart, for the rows that see them.
                uint32_t any = 0;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t bad = not_finite<T>(v[w]);
                    any |= bad;
                    v[w] &= ~bad;
                }
                if (any) atomicOr(&odd_tokens[row_of >> 5], 1u << (row_of & 31));
            }
            *reinterpret_cast<u32x4*>(to + row_of * kKeyRow + my_piece * 16) = k;
            *reinterpret_cast<u32x4*>(to + kTileTokens * kKeyRow + row_of * kValueRow + my_piece * 16) = v;
        }
    };
    // Whether some of the workgroup's rows see some of the 64 tokens and not others.
    const int last_position = place0 + static_cast<int>(a.group_size.divide(min(pair0 + kTileRows, pairs) - 1));
    const auto is_ragged = [&](int token) {
        return token + kTileTokens - 1 > sight.position || (a.window > 0 && token <= last_position - a.window);
    };

    f32x16 sum[kBlocks];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[b][i] = 0;
    float top = -__builtin_inff(), total = 0;
    const float factor = a.scale * kLog2e;
    const W weights(factor, W::kFollow ? 6 : 8);
    bool far = false;

    if (thread < 6) odd[thread >> 1][thread & 1] = 0;
    if (thread < 2 * kTileTokens) {
        char* const row = stage + thread / kTileTokens * kStage + thread % kTileTokens * kKeyRow;
        for (int piece = width / 8; piece < kPieces; ++piece) *reinterpret_cast<u32x4*>(row + piece * 16) = u32x4{0, 0, 0, 0};
    }
    int block = named_block(base);
    const Places first = places_of(block);
    uint64_t valid = valid_of(first, base);                 // of the present 64 tokens
    block = named_block(base + kTileTokens);                // of the next 64
    load(first, valid);
    bool ragged = is_ragged(base);
    __syncthreads();
    store(first, stage, ragged, odd[0]);
    __syncthreads();

    // The products of one wave's rows with 64 tokens.  kSome: not all rows see all tokens.
    const auto attend = [&](auto some, int token, int now, int turn, uint64_t valid) __attribute__((always_inline)) {
        constexpr bool kSome = decltype(some)::value;
        f32x16 score[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 16; ++i) score[h][i] = 0;
            const char* const from = stage + now + (32 * h + column) * kKeyRow + half * 16;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const Vec k = *reinterpret_cast<const Vec*>(from + s * 32);
#pragma unroll
                for (int t = 0; t < kTerms; ++t) score[h] = Matrix<T>::mul32(k, q[s][t], score[h]);
            }
        }
        const bool whole = !kSome || (valid == ~uint64_t(0) && token + kTileTokens - 1 <= low_position &&
                                      (a.window <= 0 || token > high_position - a.window));
        if (!whole) {
            int quad = 4 * half;                        // opaque: what follows from it is not kept for every stage
            asm volatile("" : "+v"(quad));
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int at = 32 * h + 8 * (i >> 2) + quad + (i & 3);
                    const bool sees = token + at <= position && token + at > after && (valid >> at & 1);
                    score[h][i] = sees ? score[h][i] : -__builtin_inff();
                }
        }
        float most = -__builtin_inff();
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 16; ++i) most = __builtin_fmaxf(most, score[h][i]);
        most = max_across_halves(most);
        // Weights may be up to 2^8 (fp16: 2^6): they keep their relative precision, and the sums are scaled again in few
        // tiles.
        if (__ballot(weights.moves(top, most))) {
            const float to = weights.moved(top, most, W::kFollow ? sum_across_halves(total) : 0);
            const float shrink = top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((top - to) * factor);
            total *= shrink;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) sum[b][i] *= shrink;
            top = to;
            far = rounds_far(top, factor);
        }
        float against = top == -__builtin_inff() ? 0.0f : __builtin_fmaf(top, factor, -W::kLift);
        if (far) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 16; ++i) score[h][i] -= top == -__builtin_inff() ? 0.0f : top;
            against = -W::kLift;
        }
        Vec p[4][kTerms];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                score[h][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[h][i], factor, -against));
                total += score[h][i];
                const int t = 2 * h + (i >> 3);
                if constexpr (kTerms == 2) two_terms(score[h][i], p[t][0], p[t][1], i & 7);
                else p[t][0][i & 7] = static_cast<T>(score[h][i]);
            }
        // V^T's operand: the four tokens that S^T left side by side, for 16 values by 16 lanes, in one
        // transposing read.
        const char* const from = stage + now + kTileTokens * kKeyRow + (4 * half + ((lane & 15) >> 2)) * kValueRow +
                                 ((lane >> 4 & 1) * 16 + (lane & 3) * 4) * 2;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                u32x4 words;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const auto four = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) short4_t*)(from + (16 * t + 8 * e) * kValueRow + b * 64));
                    const u32x2 two = bits<u32x2>(four);
                    words[2 * e] = two[0], words[2 * e + 1] = two[1];
                }
#pragma unroll
                for (int term = 0; term < kTerms; ++term)
                    sum[b] = Matrix<T>::mul32(bits<Vec>(words), p[t][term], sum[b]);
            }
        if constexpr (kSome) {
            int quad = 4 * half;
            asm volatile("" : "+v"(quad));
            const uint64_t odd_tokens = uint64_t(odd[turn][1]) << 32 | odd[turn][0];
            if (odd_tokens) {
                for (uint64_t left = odd_tokens; left; left &= left - 1) {
                    const int at = __builtin_ctzll(left);
                    float weight = 0;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            weight = 32 * h + 8 * (i >> 2) + quad + (i & 3) == at ? score[h][i] : weight;
                    weight = sum_across_halves(weight);
                    const int seen = token + at;
                    const uint32_t page = a.block_size.divide(seen);
                    const int block = table[page];
                    const char* const value = values + (block * a.layer.block_stride +
                                                        (seen - page * a.block_size.d) * a.layer.token_stride) * kBytes;
                    float scale = 1;
                    if constexpr (kEight)
                        scale = power_of(scales[block * a.layer.scale_block_stride + a.layer.scale_side_stride]);
                    const bool sees = seen <= position && seen > after;
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int d = 32 * b + 8 * (i >> 2) + quad + (i & 3);
                            if (d >= width || !sees) continue;
                            float x;
                            if constexpr (kEight)
                                x = __builtin_amdgcn_cvt_f32_fp8(static_cast<uint8_t>(value[d]), 0) * scale;
                            else x = static_cast<float>(reinterpret_cast<const T*>(value)[d]);
                            if (!(__builtin_fabsf(x) < __builtin_inff())) sum[b][i] += weight * x;
                        }
                }
            }
        }
    };

    int turn = 0;                                           // of three: whose odd tokens
    int now = 0;                                            // the buffer of these tokens
    int token = base;
    const auto one_stage = [&](auto some) __attribute__((always_inline)) {
        constexpr bool kSome = decltype(some)::value;
        const bool more = token + kTileTokens < stop;
        Places next{kNowhere, 127, 127};
        uint64_t valid_next = 0;
        if (more) {
            next = places_of(block);
            valid_next = valid_of(next, token + kTileTokens);
            block = named_block(token + 2 * kTileTokens);
            load(next, valid_next);
        }
        const int turn_next = turn == 2 ? 0 : turn + 1;
        if (thread < 2) odd[turn_next == 2 ? 0 : turn_next + 1][thread] = 0;
        if (!kSome || (!idle && token <= high_position &&
                       (a.window <= 0 || token + kTileTokens > low_position - a.window + 1)))
            attend(some, token, now, turn, valid);
        if (more) {
            ragged = is_ragged(token + kTileTokens);
            store(next, stage + kStage - now, ragged, odd[turn_next]);
            valid = valid_next;
        }
        __syncthreads();
        now = kStage - now;
        turn = turn_next;
        token += kTileTokens;
    };
    // In most stages every row sees every token: a loop of their own.
    while (token < stop) {
        while (!ragged && valid == ~uint64_t(0) && token < stop) one_stage(std::false_type{});
        if (token < stop) one_stage(std::true_type{});
    }

    total = sum_across_halves(total);
    if (!real) return;
    const int64_t index = row * a.heads + head;
    const float share = parts > 1 ? W::kDrop : over(total);
    total *= W::kDrop;
    const int64_t at_part = int64_t(blockIdx.x) * kTileRows + pair - pair0;
    float* const sums = a.tile_parts.sums + at_part * width;
    Q* const out = static_cast<Q*>(a.out) + row * a.out_token_stride + head * a.out_head_stride;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = 32 * b + 8 * i + 4 * half;
            if (d >= width) continue;
            if (parts > 1) {
                *reinterpret_cast<f32x4*>(sums + d) = f32x4{sum[b][4 * i] * share, sum[b][4 * i + 1] * share,
                                                           sum[b][4 * i + 2] * share, sum[b][4 * i + 3] * share};
            } else {
                typedef Q Four __attribute__((ext_vector_type(4)));
                Four four;
#pragma unroll
                for (int k = 0; k < 4; ++k) four[k] = static_cast<Q>(sum[b][4 * i + k] * share);
                *reinterpret_cast<Four*>(out + d) = four;
            }
        }
    if (half == 0) {
        if (parts > 1) {
            *reinterpret_cast<float2*>(a.tile_parts.totals + at_part * 2) = float2{top, total};
        } else if (a.lse) {
            a.lse[index] = top * a.scale + __builtin_logf(total);
        }
    }
}

// ----------------------------------------------------------------- parts joined

constexpr int kJoinThreads = 256, kJoinTileThreads = 64;

// `parts` parts of a row's head, `stride` heads apart, to its out.  A workgroup's threads take four values each, and
// groups of them parts in turn with a running largest score; the groups join in LDS.  The partial sums come from other
// dies' caches, about 2 us away: what counts is few steps in a row.
template <typename Q, int kThreads>
__device__ __forceinline__ void join(const Attend& a, const float* from, const float* about, int64_t stride, int parts,
                                     int row, int head) {
    const int width = a.layer.width, lanes = width >> 2;
    const int group = a.quarter_width.divide(threadIdx.x), groups = kThreads / lanes;
    const int d = (threadIdx.x - group * lanes) * 4;
    const float factor = a.scale * kLog2e;
    float top = -__builtin_inff(), total = 0;
    f32x4 x = {0, 0, 0, 0};
    if (group < groups) {
        const int64_t first = group * stride;
        from += first * width + d;
        about += first * 2;
#pragma unroll 4
        for (int c = group; c < parts; c += groups) {
            const float2 mine = *reinterpret_cast<const float2*>(about);
            const f32x4 some = *reinterpret_cast<const f32x4*>(from);
            from += groups * stride * width;
            about += groups * stride * 2;
            const float grown = __builtin_fmaxf(top, mine.x);
            const float against = grown == -__builtin_inff() ? 0.0f : grown;
            const float keep = __builtin_amdgcn_exp2f((top - against) * factor);
            const float share = __builtin_amdgcn_exp2f((mine.x - against) * factor);
            top = grown;
            total = total * keep + mine.y * share;
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = x[k] * keep + some[k] * share;
        }
    }
    __shared__ f32x4 sums[kThreads];
    __shared__ float2 tops[kThreads];
    sums[threadIdx.x] = x;
    tops[threadIdx.x] = float2{top, total};
    __syncthreads();
    if (group) return;
    for (int g = 1; g < groups; ++g) {
        const float2 mine = tops[threadIdx.x + g * lanes];
        const f32x4 some = sums[threadIdx.x + g * lanes];
        const float grown = __builtin_fmaxf(top, mine.x);
        const float against = grown == -__builtin_inff() ? 0.0f : grown;
        const float keep = __builtin_amdgcn_exp2f((top - against) * factor);
        const float share = __builtin_amdgcn_exp2f((mine.x - against) * factor);
        top = grown;
        total = total * keep + mine.y * share;
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = x[k] * keep + some[k] * share;
    }
    typedef Q Four __attribute__((ext_vector_type(4)));
    Four four;
    const float share = over(total);
#pragma unroll
    for (int k = 0; k < 4; ++k) four[k] = static_cast<Q>(x[k] * share);
    *reinterpret_cast<Four*>(static_cast<Q*>(a.out) + row * a.out_token_stride + head * a.out_head_stride + d) = four;
    if (a.lse && d == 0) a.lse[int64_t(row) * a.heads + head] = top * a.scale + __builtin_logf(total);
}

template <typename Q>
__global__ __launch_bounds__(kJoinThreads) void join_rows_kernel(Attend a) {
    const int sequence = a.all_heads.divide(blockIdx.x), head = blockIdx.x - sequence * a.heads;
    const Rows rows = rows_of(a.q, sequence, a.tokens);
    if (rows.count != 1) return;
    const int head_groups = a.layer.kv_heads / a.beside * a.head_tiles;
    const int kv_head = a.group_size.divide(head), of_key = head - kv_head * a.group;
    const int group_of = kv_head / a.beside * a.head_tiles + of_key / kHeadTile;
    const int2 info = a.row_info[int64_t(sequence) * head_groups + group_of];
    if (info.y < 2) return;                                 // written by the one workgroup that took it
    const int64_t first = (int64_t(info.x + group_of) * a.beside + kv_head % a.beside) * a.slots + of_key % kHeadTile;
    join<Q, kJoinThreads>(a, a.row_parts.sums + first * a.layer.width, a.row_parts.totals + first * 2,
            int64_t(head_groups) * a.beside * a.slots, info.y, rows.first, head);
}

template <typename Q>
__global__ __launch_bounds__(kJoinTileThreads) void join_tiles_kernel(Attend a) {
    const int row = a.all_heads.divide(blockIdx.x), head = blockIdx.x - row * a.heads;
    const int sequence = find_sequence(a.q.n_seqs, row, [&](int s) { return int64_t(a.q.query_starts[s]); });
    const Rows rows = rows_of(a.q, sequence, a.tokens);
    const int mine = row - rows.first;
    if (mine < 0 || mine >= rows.count || rows.count < a.least_rows) return;
    const int kv_head = a.group_size.divide(head), pair = mine * a.group + (head - kv_head * a.group);
    const int tile = pair / kTileRows;
    const int2 info = a.tile_info[2 * sequence], about = a.tile_info[2 * sequence + 1];
    const int64_t jobs = int64_t(about.y) * a.layer.kv_heads;           // of a part
    // Row starts that do not rise may leave a sequence without a workgroup, and its entry unwritten.
    if (info.x < 0 || info.y < 2 || about.x < 1 || tile >= about.y || info.x + jobs * info.y > a.tile_jobs) return;
    const int parts = parts_of<kTileTokens>(Split{about.x, info.y}, tile_sight(a, sequence, rows, tile * kTileRows));
    if (parts < 2) return;                                  // written by the one workgroup that took it
    const int64_t first = (info.x + int64_t(tile) * a.layer.kv_heads + kv_head) * kTileRows + pair % kTileRows;
    join<Q, kJoinTileThreads>(a, a.tile_parts.sums + first * a.layer.width, a.tile_parts.totals + first * 2,
                              jobs * kTileRows, parts, row, head);
}

// ----------------------------------------------------------------- launches

struct Plan {
    RowJobs rows;
    TileJobs tiles;
    int beside, slots, least_rows = 2;
    // Parts: of all heads, 0 where rows are whole.
    int64_t row_infos = 0, tile_infos = 0, row_jobs, tile_jobs, row_parts, tile_parts;
};

// How the rows alone are cut, as measured with 32 query heads, 8 key heads of 128 and blocks of 16 tokens, each choice
// against the other on one build.  Wider heads go by the same numbers.
//
// 8 waves side by side read a token's 8 key heads, which lie side by side, at about the same time: 64 ragged sequences
// of up to 8k tokens in e4m3 (322 MB) take 4 % longer with 4 heads beside and 37 % with one.  Few rows are better off
// with all the waves on one head: the parts are joined in LDS, and one of 32k tokens takes 20 % less.
constexpr int kFewHeads = 16;
// Jobs that the sequences' tokens are cut into: in e4m3 no more than the chip holds at once, two workgroups a CU up to
// width 128 (one row over 32k tokens takes 13 % longer with 450 asked for, the 64 ragged ones 14 % with 512 asked for and
// some 530 made).  A 16-bit cache's jobs are longer, and about twice as many are better (500: 12 % longer; no more than
// 1000: 4 %).
constexpr int kRoomE4m3 = 512, kRoom16 = 1000;
// Tiles of a wave up to which a row is not cut, the join being 4 to 7 us, and of a part at least.
constexpr int kWholeTurns = 5, kLeastTurns = 2;

// Tiles whose jobs are fewer than the chip holds at once (two workgroups a CU up to width 128; wider ones hold one, and
// go in two rounds) are cut into no more than that, where it comes out: with 12 sequences of up to 7700 tokens and 693
// rows (16 heads over 8 of 128, e4m3) parts of one length by the longest sequence's, as for three rounds, took 17 %
// longer, the last round being nearly empty.  So are up to four times as many where a sequence's rows fill less than a
// tile, so that its tokens alone make its work: 64 sequences of up to 8k tokens with 1 to 3 rows each (32 heads over 8)
// take 2.6 times as long whole.  A prompt's tiles are better whole, the later ones first (2048 tokens: 27 % longer cut).
constexpr int kTileRoom = 512, kMostCut = 4 * kTileRoom;

Plan plan_of(int64_t tokens, int n_seqs, bool ragged, int heads, int kv_heads, bool eight, int64_t max_length,
             int64_t window) {
    int64_t longest = window > 0 ? std::min(window, max_length) : max_length;
    const int64_t group = heads / kv_heads, head_tiles = (group + kHeadTile - 1) / kHeadTile;
    Plan plan{};
    plan.beside = 1;
    if (n_seqs * int64_t(kv_heads) >= kFewHeads)
        while (plan.beside < kWaves && kv_heads % (2 * plan.beside) == 0) plan.beside *= 2;
    plan.slots = static_cast<int>(std::min<int64_t>(group, kHeadTile));
    const int64_t row_jobs = n_seqs * head_tiles * (kv_heads / plan.beside);
    const int64_t tiles = std::max<int64_t>((longest + kTile - 1) / kTile + 1, 1);
    const int64_t in_turn = kWaves / plan.beside;
    const int64_t least = kLeastTurns * in_turn, whole = kWholeTurns * in_turn;
    const int room = eight ? kRoomE4m3 : kRoom16;
    plan.rows = RowJobs{0, 1 << 24, 1, room, eight};
    plan.row_jobs = row_jobs;
    if (tiles > whole && n_seqs <= kEvenSeqs) {
        plan.rows.even = 1;
        plan.rows.chunk = static_cast<int>(least);
        plan.row_jobs += room;
        plan.row_parts = plan.row_jobs * plan.beside * plan.slots;
    } else if (tiles > whole) {
        plan.rows.chunk = static_cast<int>(std::min<int64_t>(std::max(least, tiles * row_jobs / (2 * room)), 1 << 24));
        plan.rows.chunks = static_cast<int>((tiles + plan.rows.chunk - 1) / plan.rows.chunk);
        plan.row_jobs *= plan.rows.chunks;
        if (plan.rows.chunks > 1) plan.row_parts = plan.row_jobs * plan.beside * plan.slots;
    }
    if (plan.row_parts) plan.row_infos = row_jobs;
    if (ragged && n_seqs == 1 && tokens > 1) {
        // A prompt or chunk alone: tiles take it, also where all its rows but one are padding, and there is no launch
        // that looks for rows alone (10 us with its join).
        plan.row_jobs = plan.row_parts = plan.row_infos = 0;
        plan.least_rows = 1;
    }
    if (ragged) {
        const int64_t full_tiles = tokens * group / kTileRows;
        plan.tile_jobs = (full_tiles + n_seqs) * kv_heads;
        // A tile's rows see from the first's window to the last's own token.
        longest = std::min(max_length, longest + (kTileRows + group - 1) / group);
        if (plan.tile_jobs < (full_tiles < n_seqs ? kMostCut : kTileRoom) && n_seqs <= kTileSeqs &&
            longest > kLeastStages * kTileTokens) {
            plan.tiles = TileJobs{1, kTileRoom};
            plan.tile_jobs += kTileRoom;
            plan.tile_parts = plan.tile_jobs * kTileRows;
            plan.tile_infos = 2 * int64_t(n_seqs);
        }
    }
    return plan;
}

size_t bytes_of(const Plan& plan, int width) {
    return static_cast<size_t>(plan.row_parts + plan.tile_parts) * (width + 2) * sizeof(float) +
           static_cast<size_t>(plan.row_infos + plan.tile_infos) * sizeof(int2);
}

template <typename Q, bool kEight, int kJ>
void launch_rows_of(const Attend& a, unsigned grid, unsigned lds, hipStream_t stream) {
    const auto kernel = a.layer.block_size % 16     ? attend_row_kernel<Q, kEight, kJ, false, false>
                        : a.layer.width == 16 * kJ ? attend_row_kernel<Q, kEight, kJ, true, true>
                                                   : attend_row_kernel<Q, kEight, kJ, true, false>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kWaves * 64), lds, stream, a);
}

template <typename Q, bool kEight>
void launch_rows(const Attend& a, unsigned grid, unsigned lds, hipStream_t stream) {
    if (a.layer.width <= 64) launch_rows_of<Q, kEight, 4>(a, grid, lds, stream);
    else if (a.layer.width <= 128) launch_rows_of<Q, kEight, 8>(a, grid, lds, stream);
    else launch_rows_of<Q, kEight, 16>(a, grid, lds, stream);
}

template <typename Q, bool kEight, bool kWhole>
void launch_tiles_of(const Attend& a, unsigned grid, hipStream_t stream) {
    const auto kernel = a.layer.width <= 64    ? attend_tile_kernel<Q, kEight, 64, kWhole>
                        : a.layer.width <= 96  ? attend_tile_kernel<Q, kEight, 96, kWhole>
                        : a.layer.width <= 128 ? attend_tile_kernel<Q, kEight, 128, kWhole>
                        : a.layer.width <= 192 ? attend_tile_kernel<Q, kEight, 192, kWhole>
                                               : attend_tile_kernel<Q, kEight, 256, kWhole>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kTileWaves * 64), 0, stream, a);
}

template <typename Q, bool kEight>
void launch_tiles(const Attend& a, unsigned grid, hipStream_t stream) {
    if (a.layer.block_size % 16) launch_tiles_of<Q, kEight, false>(a, grid, stream);
    else launch_tiles_of<Q, kEight, true>(a, grid, stream);
}

unsigned checked_grid(int64_t groups, int threads) {
    require(groups * threads < (int64_t(1) << 32), "attend: too many rows for one launch");
    return static_cast<unsigned>(groups);
}

template <typename Q>
void launch_attend(const Attend& a, const Plan& plan, hipStream_t stream) {
    const bool eight = a.layer.type == KVSNAP_E4M3;
    if (plan.tile_jobs) {
        const unsigned grid = checked_grid(plan.tile_jobs, kTileWaves * 64);
        if (eight) launch_tiles<Q, true>(a, grid, stream);
        else launch_tiles<Q, false>(a, grid, stream);
        check_launched("attend's tiles");
    }
    if (plan.row_jobs) {
        const unsigned grid = checked_grid(plan.row_jobs, kWaves * 64);
        const unsigned lds = 4u * (kWaves * std::min(kHeadTile, a.group) * a.layer.width + 2 * kWaves * kHeadTile);
        if (eight) launch_rows<Q, true>(a, grid, lds, stream);
        else launch_rows<Q, false>(a, grid, lds, stream);
        check_launched("attend's rows");
    }
    if (plan.row_parts) {
        hipLaunchKernelGGL(join_rows_kernel<Q>, dim3(checked_grid(int64_t(a.q.n_seqs) * a.heads, kJoinThreads)),
                           dim3(kJoinThreads), 0, stream, a);
        check_launched("attend's joins");
    }
    if (plan.tile_parts) {
        hipLaunchKernelGGL(join_tiles_kernel<Q>, dim3(checked_grid(int64_t(a.tokens) * a.heads, kJoinTileThreads)),
                           dim3(kJoinTileThreads), 0, stream, a);
        check_launched("attend's joins");
    }
}

}  // namespace

extern "C" {

size_t kvsnap_attend_workspace_bytes(const kvsnap_paged_layer* layer, int64_t tokens, int n_seqs, int ragged, int heads,
                                     int64_t max_length, int64_t window) {
    if (!layer || tokens <= 0 || n_seqs <= 0 || heads <= 0 || layer->kv_heads <= 0 || heads % layer->kv_heads) return 0;
    return bytes_of(plan_of(tokens, n_seqs, ragged, heads, layer->kv_heads, layer->type == KVSNAP_E4M3, max_length,
                            std::min<int64_t>(window, 1 << 30)),
                    layer->width);
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
        require(tokens * heads < (int64_t(1) << 31), "attend: too many rows for one launch");
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
        a.window = static_cast<int>(std::min<int64_t>(window, 1 << 30));
        const int64_t named = int64_t(sequences->table_width) * layer->block_size;
        const Plan plan = plan_of(tokens, sequences->n_seqs, sequences->query_starts != nullptr, heads,
                                  layer->kv_heads, layer->type == KVSNAP_E4M3, std::min(max_length, named), a.window);
        a.head_tiles = (a.group + kHeadTile - 1) / kHeadTile;
        a.beside = plan.beside, a.slots = plan.slots, a.least_rows = plan.least_rows;
        a.block_size = Divider::of(layer->block_size);
        a.group_size = Divider::of(a.group);
        a.all_heads = Divider::of(heads);
        const int64_t element = layer->type == KVSNAP_E4M3 ? 1 : 2;
        a.block_pieces = static_cast<uint32_t>(layer->block_stride * element / 16);
        a.token_pieces = static_cast<uint32_t>(layer->token_stride * element / 16);
        a.stage_pages = kTileTokens / layer->block_size, a.stage_slots = kTileTokens % layer->block_size;
        a.quarter_width = Divider::of(layer->width / 4);
        a.rows = plan.rows, a.tiles = plan.tiles;
        float* const room = static_cast<float*>(workspace);
        const int64_t parts = plan.row_parts + plan.tile_parts;
        a.row_parts = Parts{room, room + parts * layer->width};
        a.tile_parts = Parts{room + plan.row_parts * layer->width, a.row_parts.totals + plan.row_parts * 2};
        int2* const infos = reinterpret_cast<int2*>(room + parts * (layer->width + 2));
        if (plan.row_infos) a.row_info = infos;
        if (plan.tile_infos) a.tile_info = infos + plan.row_infos;
        a.tile_jobs = static_cast<int>(plan.tile_jobs);
        require(workspace_bytes >= bytes_of(plan, layer->width), "attend: the workspace is too small");
        require(parts == 0 || (workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                "attend: the workspace must be 16-byte aligned device memory");
        const auto launch = type == KVSNAP_BF16 ? launch_attend<__bf16> : launch_attend<_Float16>;
        launch(a, plan, reinterpret_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
