// Rotating queries and keys by their positions, and a step's keys and values into a layer's paged cache
// (include/kvsnap_attention.h).
//
// A pair (a, b) of a head's values becomes (a cos - b sin, b cos + a sin) of its position's angle, in fp32 from the
// inputs' type and rounded once, to the output's.  Nothing here is more than one pass over the data, so memory is the
// bound: a lane takes 16 values of one head (two 16-byte loads, eight pairs, the 64 bytes of their angles), so a pair
// never leaves its lane.  Turning 16,384 tokens of 32 heads of 128 by three axes (277 MB in and out) takes 52 us (a kernel
// trace's), 5.3 TB/s, as fast as a large copy goes on this card (5.2 to 5.4).
#include "launch.h"
#include "paged.h"

#include <initializer_list>

namespace {

using namespace kvsnap;

constexpr int kLanes = 256;  // 4 waves a workgroup
constexpr int kUnit = 16;    // values of a lane

// ----------------------------------------------------------------- values

__device__ __forceinline__ void load8(const __bf16* p, float* v) {
    const bf16x8 x = *reinterpret_cast<const bf16x8*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(x[i]);
}
__device__ __forceinline__ void load8(const _Float16* p, float* v) {
    const half8_t x = *reinterpret_cast<const half8_t*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(x[i]);
}
__device__ __forceinline__ void load8(const float* p, float* v) {
    const f32x4 x = reinterpret_cast<const f32x4*>(p)[0], y = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = x[i], v[4 + i] = y[i];
}
__device__ __forceinline__ void store8(__bf16* p, const float* v) {
    bf16x8 x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<__bf16>(v[i]);
    *reinterpret_cast<bf16x8*>(p) = x;
}
__device__ __forceinline__ void store8(_Float16* p, const float* v) {
    half8_t x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<_Float16>(v[i]);
    *reinterpret_cast<half8_t*>(p) = x;
}
__device__ __forceinline__ void store8(float* p, const float* v) {
    reinterpret_cast<f32x4*>(p)[0] = f32x4{v[0], v[1], v[2], v[3]};
    reinterpret_cast<f32x4*>(p)[1] = f32x4{v[4], v[5], v[6], v[7]};
}

// Four values to e4m3, to the nearest, ties to even; what is not finite becomes NaN.
__device__ __forceinline__ uint32_t pack_e4m3(const float* v) {
    int word = 0;
    word = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], word, false);
    word = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], word, true);
    return static_cast<uint32_t>(word);
}
__device__ __forceinline__ void unpack_e4m3(uint32_t word, float* v) {
    const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(word, false), high = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
    v[0] = low[0], v[1] = low[1], v[2] = high[0], v[3] = high[1];
}

// ----------------------------------------------------------------- rotation

// Where a unit's two runs of eight values start in its head.  Pairs j and j + pairs of units below pairs / 8 are the
// same elements of the two runs; adjacent pairs and the values past the turned ones lie in one run of sixteen.
__device__ __forceinline__ int second_run(const kvsnap_rotation& r, int unit) {
    return !r.interleaved && unit * 8 < r.pairs ? unit * 8 + r.pairs : unit * kUnit + 8;
}
__device__ __forceinline__ int first_run(const kvsnap_rotation& r, int unit) {
    return !r.interleaved && unit * 8 < r.pairs ? unit * 8 : unit * kUnit;
}

__device__ __forceinline__ const float* angle_row(const kvsnap_rotation& r, int axis, int64_t token, int64_t counted) {
    int64_t at = counted;
    if (r.positions) {
        const int64_t index = axis * r.axis_stride + token;
        at = r.narrow ? static_cast<const int32_t*>(r.positions)[index]
                      : static_cast<const int64_t*>(r.positions)[index];
    }
    return at >= 0 && at < r.rows ? r.angles + at * r.pairs * 2 : nullptr;
}

// Turns a unit's pairs in place: v holds its two runs.  `token` is the row in the positions, `counted` its position
// where there are none.
__device__ __forceinline__ void turn(const kvsnap_rotation& r, int unit, int64_t token, int64_t counted, float* v) {
    if (!r.angles || unit * 8 >= r.pairs) return;
    float angle[16];  // cosine and sine of each pair
    const uint32_t axes = r.axes[unit];
    if (axes == (axes & 3) * 0x5555u) {
        const float* row = angle_row(r, axes & 3, token, counted);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f32x4 some = {__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
            if (row) some = reinterpret_cast<const f32x4*>(row + unit * 16)[i];
#pragma unroll
            for (int k = 0; k < 4; ++k) angle[4 * i + k] = some[k];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float* row = angle_row(r, (axes >> (2 * j)) & 3, token, counted);
            angle[2 * j] = row ? row[unit * 16 + 2 * j] : __builtin_nanf("");
            angle[2 * j + 1] = row ? row[unit * 16 + 2 * j + 1] : __builtin_nanf("");
        }
    }
    float turned[kUnit];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float cos = angle[2 * j], sin = r.inverse ? -angle[2 * j + 1] : angle[2 * j + 1];
        const float a = r.interleaved ? v[2 * j] : v[j], b = r.interleaved ? v[2 * j + 1] : v[8 + j];
        const float x = a * cos - b * sin, y = b * cos + a * sin;
        // Both places are written by select, so the arrays stay in registers.
        if (r.interleaved) turned[2 * j] = x, turned[2 * j + 1] = y;
        else turned[j] = x, turned[8 + j] = y;
    }
#pragma unroll
    for (int i = 0; i < kUnit; ++i) v[i] = turned[i];
}

// One unit of a head, as it comes and as it goes.
template <typename T>
__device__ __forceinline__ void load_unit(const kvsnap_rotation& r, const T* in, int unit, float* v) {
    load8(in + first_run(r, unit), v);
    load8(in + second_run(r, unit), v + 8);
}
template <typename T>
__device__ __forceinline__ void store_unit(const kvsnap_rotation& r, T* out, int unit, const float* v) {
    store8(out + first_run(r, unit), v);
    store8(out + second_run(r, unit), v + 8);
}

template <typename T>
struct Strided {
    T* at;
    int64_t token_stride, head_stride;

    __device__ __forceinline__ T* row(int64_t token, int head) const {
        return at + token * token_stride + head * head_stride;
    }
};

template <typename T>
__global__ __launch_bounds__(kLanes) void rotate_kernel(Strided<const T> x, Strided<T> out, uint32_t items,
                                                        Divider per_token, Divider units, kvsnap_rotation r) {
    const uint32_t item = blockIdx.x * kLanes + threadIdx.x;
    if (item >= items) return;
    const uint32_t token = per_token.divide(item), rest = item - token * per_token.d;
    const uint32_t head = units.divide(rest), unit = rest - head * units.d;
    float v[kUnit];
    load_unit(r, x.row(token, head), unit, v);
    turn(r, unit, token, token, v);
    store_unit(r, out.row(token, head), unit, v);
}

// ----------------------------------------------------------------- append

template <typename T>
struct Step {
    Strided<const T> key, value, query;
    Strided<T> query_out;
    int tokens, heads;
    uint32_t query_items, query_groups;  // workgroups [0, query_groups) turn the queries
    uint32_t items;                      // of keys and values: units, or a wave's jobs for an e4m3 cache
    Divider units, query_per_token, kv_per_token, block_size;
};

// The sequence of each lane's row and the row's position there, or a negative position for a row that is padding.
// The wave searches for its first row's; a lane goes on from there by steps that double, and back by halves: a wave's rows
// are few, but between two of them may lie all the sequences of a padded batch that have none.
__device__ __forceinline__ int locate(const kvsnap_sequences& q, int row, int tokens, int& sequence) {
    sequence = row;
    if (q.query_starts) {
        const int first = __builtin_amdgcn_readfirstlane(row);
        sequence = find_sequence(q.n_seqs, first, [&](int s) { return int64_t(q.query_starts[s]); });
        int step = 1;
        for (; step < q.n_seqs - sequence && q.query_starts[sequence + step] <= row; step *= 2) sequence += step;
        for (int high = min(step, q.n_seqs - sequence); high > 1;) {
            const int half = high >> 1;
            const bool passed = q.query_starts[sequence + half] <= row;
            if (passed) sequence += half;
            high = passed ? high - half : half;
        }
    }
    const Rows rows = rows_of(q, sequence, tokens);
    const int i = row - rows.first;
    return i >= 0 && i < rows.count ? length_of(q, sequence) - rows.count + i : -1;
}

template <typename T>
__device__ __forceinline__ void append_query(const Step<T>& step, const kvsnap_sequences& q,
                                             const kvsnap_rotation& r) {
    const uint32_t item = min(blockIdx.x * kLanes + threadIdx.x, step.query_items - 1);
    const uint32_t token = step.query_per_token.divide(item), rest = item - token * step.query_per_token.d;
    const uint32_t head = step.units.divide(rest), unit = rest - head * step.units.d;
    float v[kUnit];
    load_unit(r, step.query.row(token, head), unit, v);     // under way while the row's position is looked for
    int sequence;
    const int at = locate(q, token, step.tokens, sequence);
    if (at < 0 || blockIdx.x * kLanes + threadIdx.x >= step.query_items) return;
    turn(r, unit, token, at, v);
    store_unit(r, step.query_out.row(token, head), unit, v);
}

// A 16-bit cache: each unit of a key or value to its slot, and the queries beside them in the same launch.  Two 8k prompts
// of 32 heads over 8 of 128 (411 MB) take 84 us, 4.9 TB/s: the memory's rate for a copy, less the scattered slots.  A
// decode step's 0.02 to 1.5 MB take 5.4 us, 4.4 of them the launch.
template <typename T>
__global__ __launch_bounds__(kLanes) void append_kernel(Step<T> step, kvsnap_paged_layer layer, kvsnap_sequences q,
                                                        kvsnap_rotation r) {
    if (blockIdx.x < step.query_groups) return append_query(step, q, r);
    const uint32_t index = (blockIdx.x - step.query_groups) * kLanes + threadIdx.x;
    const uint32_t item = min(index, step.items - 1);
    const uint32_t token = step.kv_per_token.divide(item), rest = item - token * step.kv_per_token.d;
    const uint32_t side_head = step.units.divide(rest), unit = rest - side_head * step.units.d;
    const bool is_value = side_head >= static_cast<uint32_t>(layer.kv_heads);
    const uint32_t head = is_value ? side_head - layer.kv_heads : side_head;
    float v[kUnit] = {};
    u32x4 copied[2] = {};
    if (is_value) {
        const u32x4* const from = reinterpret_cast<const u32x4*>(step.value.row(token, head) + unit * kUnit);
        copied[0] = from[0], copied[1] = from[1];
    } else {
        load_unit(r, step.key.row(token, head), unit, v);
    }
    int sequence;
    const int at = locate(q, token, step.tokens, sequence);
    if (at < 0 || index >= step.items) return;
    const uint32_t page = step.block_size.divide(at), slot = at - page * step.block_size.d;
    if (page >= static_cast<uint32_t>(q.table_width)) return;
    const int64_t block = q.block_tables[sequence * q.table_stride + page];
    if (!is_value) turn(r, unit, token, at, v);
    if (block < 0 || block >= layer.blocks) return;
    T* const cache = static_cast<T*>(is_value ? layer.value : layer.key) + block * layer.block_stride +
                     slot * layer.token_stride + head * layer.head_stride;
    if (is_value) {
        reinterpret_cast<u32x4*>(cache + unit * kUnit)[0] = copied[0];
        reinterpret_cast<u32x4*>(cache + unit * kUnit)[1] = copied[1];
    } else {
        store_unit(r, cache, unit, v);
    }
}

// The e8m0 byte of the least power of two s with top <= 448 s (448 = 1.75 * 2^8 is e4m3's largest value), from
// top's exponent and mantissa, so that it is exact; at least 1 (2^-126).
__device__ __forceinline__ int scale_for(float top) {
    const uint32_t word = bits<uint32_t>(top);
    const int e = static_cast<int>(word >> 23) - 8 + ((word & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, 1);
}

// An e4m3 cache: a wave takes one head's keys or values in one block, so that the block's scale is one wave's to
// decide, 64 / (width / 16) rows at a time.  Blocks of up to kKeep such passes (16 tokens of 128 are two) stay in
// registers between looking for their largest value and being written; longer ones are read again.  Loads that do not
// follow from one another are under way together: the table's entry, the rows, their angles.  Ragged chunks (3.8 MB) take
// 12 us, a chain of loads: row starts, lengths, rows and angles, the block's scale, its filled slots (40 % longer with each
// kept row loaded and turned before the next).  The last two follow from the table's entry alone, and wait behind the
// rows' largest value only because they are asked for there.  Two 8k prompts (377 MB) take 91 us, 4.1 TB/s.
template <typename T, int kKeep>
__global__ __launch_bounds__(kLanes) void append_e4m3_kernel(Step<T> step, kvsnap_paged_layer layer,
                                                             kvsnap_sequences q, kvsnap_rotation r) {
    if (blockIdx.x < step.query_groups) return append_query(step, q, r);
    const uint32_t job = __builtin_amdgcn_readfirstlane((blockIdx.x - step.query_groups) * (kLanes / 64) +
                                                        (threadIdx.x >> 6));
    if (job >= step.items) return;
    const uint32_t work = step.kv_per_token.divide(job), side_head = job - work * step.kv_per_token.d;
    const bool is_value = side_head >= static_cast<uint32_t>(layer.kv_heads);
    const int head = is_value ? side_head - layer.kv_heads : side_head, size = layer.block_size;
    // Sequence s has shares from query_starts[s] / size + 2 s on: n rows touch at most n / size + 2 blocks.
    int sequence = work;
    int64_t share = work;
    const auto shares = [&](int s) {
        return int64_t(step.block_size.divide(min(max(q.query_starts[s], 0), step.tokens))) + 2 * s;
    };
    if (q.query_starts) {
        sequence = find_sequence(q.n_seqs, work, shares);
        share = shares(sequence);
    }
    const Rows rows = rows_of(q, sequence, step.tokens);
    if (!rows.count) return;
    const int length = length_of(q, sequence), first = length - rows.count;
    const int page = step.block_size.divide(max(first, 0)) + static_cast<int>(work - share);
    if (work < share || page >= q.table_width) return;
    const int begin = max(first, page * size), end = min(length, (page + 1) * size);
    if (begin >= end) return;
    const int64_t block = q.block_tables[sequence * q.table_stride + page];

    const int lane = threadIdx.x & 63;
    const int units = step.units.d, per_pass = 64 / units;
    const int row = step.units.divide(lane), unit = lane - row * units;
    const int run0 = is_value ? unit * kUnit : first_run(r, unit);
    const int run1 = is_value ? unit * kUnit + 8 : second_run(r, unit);
    const int low = row < per_pass ? begin + row : end;     // lanes past the last whole row take none
    const auto load = [&](int at, float* v) {
        const int64_t token = rows.first + at - first;
        const T* const from = is_value ? step.value.row(token, head) : step.key.row(token, head);
        load8(from + run0, v);
        load8(from + run1, v + 8);
    };
    const auto turned = [&](int at, float* v) {
        if (!is_value) turn(r, unit, rows.first + at - first, at, v);
    };
    float top = 0;
    const auto look = [&](const float* v) {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) {
            const float size_of = __builtin_fabsf(v[i]);
            top = size_of < __builtin_inff() ? __builtin_fmaxf(top, size_of) : top;
        }
    };
    float kept[kKeep > 0 ? kKeep : 1][kUnit];
    if constexpr (kKeep > 0) {
#pragma unroll
        for (int k = 0; k < kKeep; ++k)
            if (low + k * per_pass < end) load(low + k * per_pass, kept[k]);
#pragma unroll
        for (int k = 0; k < kKeep; ++k)
            if (low + k * per_pass < end) {
                turned(low + k * per_pass, kept[k]);
                look(kept[k]);
            }
    } else {
        for (int at = low; at < end; at += per_pass) {
            float v[kUnit];
            load(at, v);
            turned(at, v);
            look(v);
        }
    }
    if (block < 0 || block >= layer.blocks) return;
    uint8_t* const held = layer.scales + block * layer.scale_block_stride + head * layer.scale_head_stride +
                          (is_value ? layer.scale_side_stride : 0);
    uint8_t* const cache = static_cast<uint8_t*>(is_value ? layer.value : layer.key) + block * layer.block_stride +
                           head * layer.head_stride;
    const int filled = begin - page * size;
    const int before = filled > 0 ? *held : 0;
#pragma unroll
    for (int step_of = 1; step_of < 64; step_of <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, step_of));
    const int scale = max(scale_for(top), before);
    if (filled > 0 && scale > before) {
        // The slots before the new ones, rounded again: a power of two only costs the bits that fall under e4m3's least
        // value.
        for (int slot = row; slot < filled && row < per_pass; slot += per_pass) {
            u32x4* const words = reinterpret_cast<u32x4*>(cache + slot * layer.token_stride + unit * kUnit);
            u32x4 old = *words;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[4];
                unpack_e4m3(old[i], v);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = __builtin_amdgcn_ldexpf(v[k], before - scale);
                old[i] = pack_e4m3(v);
            }
            *words = old;
        }
    }
    const auto write = [&](int at, float* v) {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) v[i] = __builtin_amdgcn_ldexpf(v[i], 127 - scale);
        uint8_t* const to = cache + (at - page * size) * layer.token_stride;
        *reinterpret_cast<u32x2*>(to + run0) = u32x2{pack_e4m3(v), pack_e4m3(v + 4)};
        *reinterpret_cast<u32x2*>(to + run1) = u32x2{pack_e4m3(v + 8), pack_e4m3(v + 12)};
    };
    if constexpr (kKeep > 0) {
#pragma unroll
        for (int k = 0; k < kKeep; ++k)
            if (low + k * per_pass < end) write(low + k * per_pass, kept[k]);
    } else {
        for (int at = low; at < end; at += per_pass) {
            float v[kUnit];
            load(at, v);
            turned(at, v);
            write(at, v);
        }
    }
    if (lane == 0) *held = static_cast<uint8_t>(scale);
}

// ----------------------------------------------------------------- launches

bool aligned(const void* p, std::initializer_list<int64_t> strides, int64_t element) {
    bool fits = reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (int64_t stride : strides) fits = fits && stride * element % 16 == 0;
    return fits;
}

kvsnap_rotation checked_rotation(const kvsnap_rotation* rotation, int width) {
    kvsnap_rotation none{};
    if (!rotation || !rotation->angles) return none;
    require(rotation->pairs > 0 && rotation->pairs % 8 == 0 && 2 * rotation->pairs <= width,
            "rotation: the pairs must be a multiple of 8 and fit the width");
    require(rotation->rows >= 0, "rotation: negative rows");
    require(reinterpret_cast<uintptr_t>(rotation->angles) % 16 == 0, "rotation: angles must be 16-byte aligned");
    return *rotation;
}

uint32_t counted_items(int64_t a, int64_t b, int64_t c) {
    const __int128 n = __int128(a) * b * c;
    require(n < (int64_t(1) << 31), "too many values for one launch");
    return static_cast<uint32_t>(n);
}

unsigned groups_of(uint32_t items, int each) { return (items + each - 1) / each; }

template <typename T>
void launch_rotate(const void* x, int64_t x_token_stride, int64_t x_head_stride, void* out, int64_t out_token_stride,
                   int64_t out_head_stride, uint32_t items, int heads, int width, const kvsnap_rotation& r,
                   hipStream_t stream) {
    hipLaunchKernelGGL(rotate_kernel<T>, dim3(groups_of(items, kLanes)), dim3(kLanes), 0, stream,
                       (Strided<const T>{static_cast<const T*>(x), x_token_stride, x_head_stride}),
                       (Strided<T>{static_cast<T*>(out), out_token_stride, out_head_stride}), items,
                       Divider::of(heads * (width / kUnit)), Divider::of(width / kUnit), r);
    check_launched("rotate");
}

template <typename T>
void launch_append(const kvsnap_paged_layer& layer, const kvsnap_sequences& q, const kvsnap_rotation& r,
                   const void* key, int64_t key_token_stride, int64_t key_head_stride, const void* value,
                   int64_t value_token_stride, int64_t value_head_stride, const void* query, int64_t query_token_stride,
                   int64_t query_head_stride, void* query_out, int64_t out_token_stride, int64_t out_head_stride,
                   int64_t tokens, int heads, hipStream_t stream) {
    const int units = layer.width / kUnit;
    Step<T> step{};
    step.key = {static_cast<const T*>(key), key_token_stride, key_head_stride};
    step.value = {static_cast<const T*>(value), value_token_stride, value_head_stride};
    step.query = {static_cast<const T*>(query), query_token_stride, query_head_stride};
    step.query_out = {static_cast<T*>(query_out), out_token_stride, out_head_stride};
    step.tokens = static_cast<int>(tokens);
    step.heads = heads;
    step.units = Divider::of(units);
    step.block_size = Divider::of(layer.block_size);
    if (query) {
        step.query_items = counted_items(tokens, heads, units);
        step.query_groups = groups_of(step.query_items, kLanes);
        step.query_per_token = Divider::of(heads * units);
    }
    if (layer.type == KVSNAP_E4M3) {
        const int64_t work = q.query_starts ? tokens / layer.block_size + 2 * int64_t(q.n_seqs) : tokens;
        step.items = counted_items(work, layer.kv_heads, 2);
        step.kv_per_token = Divider::of(2 * layer.kv_heads);
        // Passes over a block, or over the one row that a sequence adds where there are no query_starts.
        const int passes = q.query_starts ? (layer.block_size + 64 / units - 1) / (64 / units) : 1;
        const auto kernel = passes == 1   ? append_e4m3_kernel<T, 1>
                            : passes == 2 ? append_e4m3_kernel<T, 2>
                            : passes <= 4 ? append_e4m3_kernel<T, 4>
                                          : append_e4m3_kernel<T, 0>;
        hipLaunchKernelGGL(kernel, dim3(step.query_groups + groups_of(step.items, kLanes / 64)), dim3(kLanes), 0,
                           stream, step, layer, q, r);
    } else {
        step.items = counted_items(tokens, 2 * int64_t(layer.kv_heads), units);
        step.kv_per_token = Divider::of(2 * layer.kv_heads * units);
        hipLaunchKernelGGL(append_kernel<T>, dim3(step.query_groups + groups_of(step.items, kLanes)), dim3(kLanes), 0,
                           stream, step, layer, q, r);
    }
    check_launched("append");
}

}  // namespace

extern "C" {

int kvsnap_rotate(const void* x, int64_t x_token_stride, int64_t x_head_stride, void* out, int64_t out_token_stride,
                  int64_t out_head_stride, int64_t tokens, int heads, int width, int type,
                  const kvsnap_rotation* rotation, uintptr_t stream) {
    return guarded([&] {
        require(tokens >= 0 && heads >= 0, "rotate: negative size");
        require(width > 0 && width % kUnit == 0 && width <= 256, "rotate: the width must be a multiple of 16 up to 256");
        if (tokens == 0 || heads == 0) return;
        require(x && out && rotation && rotation->angles, "rotate needs device pointers");
        const int64_t element = type == KVSNAP_FP32 ? 4 : 2;
        require(aligned(x, {x_token_stride, x_head_stride}, element) &&
                    aligned(out, {out_token_stride, out_head_stride}, element),
                "rotate: rows and heads must be 16-byte aligned");
        const kvsnap_rotation r = checked_rotation(rotation, width);
        const uint32_t items = counted_items(tokens, heads, width / kUnit);
        const auto launch = type == KVSNAP_BF16   ? launch_rotate<__bf16>
                            : type == KVSNAP_FP16 ? launch_rotate<_Float16>
                            : type == KVSNAP_FP32 ? launch_rotate<float>
                                                  : nullptr;
        require(launch, "rotate: values must be bf16, fp16 or fp32");
        launch(x, x_token_stride, x_head_stride, out, out_token_stride, out_head_stride, items, heads, width, r,
               reinterpret_cast<hipStream_t>(stream));
    });
}

int kvsnap_append(const kvsnap_paged_layer* layer, const kvsnap_sequences* sequences, const kvsnap_rotation* rotation,
                  const void* key, int64_t key_token_stride, int64_t key_head_stride, const void* value,
                  int64_t value_token_stride, int64_t value_head_stride, const void* query, int64_t query_token_stride,
                  int64_t query_head_stride, void* query_out, int64_t out_token_stride, int64_t out_head_stride,
                  int64_t tokens, int heads, int type, uintptr_t stream) {
    return guarded([&] {
        require(layer && sequences, "append needs a layer and its sequences");
        check_layer(*layer);
        check_sequences(*sequences, *layer);
        require(tokens >= 0 && heads >= 0, "append: negative size");
        require(tokens < (int64_t(1) << 31), "append: too many tokens");
        if (tokens == 0 || sequences->n_seqs == 0) return;
        require(sequences->query_starts || tokens == sequences->n_seqs,
                "append: without query_starts every sequence has one row");
        require(type == KVSNAP_BF16 || type == KVSNAP_FP16, "append: keys and values must be bf16 or fp16");
        require(layer->type == KVSNAP_E4M3 || layer->type == type, "append: a 16-bit cache must have the keys' type");
        require(key && value && (!query || query_out), "append needs device pointers");
        require(aligned(key, {key_token_stride, key_head_stride}, 2) &&
                    aligned(value, {value_token_stride, value_head_stride}, 2) &&
                    (!query || (aligned(query, {query_token_stride, query_head_stride}, 2) &&
                                aligned(query_out, {out_token_stride, out_head_stride}, 2))),
                "append: rows and heads must be 16-byte aligned");
        const kvsnap_rotation r = checked_rotation(rotation, layer->width);
        const auto launch = type == KVSNAP_BF16 ? launch_append<__bf16> : launch_append<_Float16>;
        launch(*layer, *sequences, r, key, key_token_stride, key_head_stride, value, value_token_stride,
               value_head_stride, heads ? query : nullptr, query_token_stride, query_head_stride, query_out,
               out_token_stride, out_head_stride, tokens, heads, reinterpret_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
