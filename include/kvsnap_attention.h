/*
 * Operators over one layer's paged KV cache (gfx950), built into
 * kvsnap_amd/_native/libkvsnap_hip.so beside the snapshot kernels: rotating
 * queries and keys by their positions, appending keys and values to the
 * cache, and attention over it.  No counterpart in the reference, whose
 * engine brings its own.
 *
 * As in kvsnap_kernels.h: buffers are device addresses, every entry point
 * launches on `stream` on the current device, returns 0 once the launch is
 * queued and -1 with kvsnap_cuda_error() set if the arguments are refused or
 * the launch fails.  Nothing is allocated, nothing synchronizes, and no
 * memory is touched but what the arguments name, so launches may be captured.
 *
 * A layer's cache is blocks of `block_size` token slots, `kv_heads` heads of
 * `width` values for K and for V, where value d of head h in slot t of block
 * b is at key (or value) + b * block_stride + t * token_stride + h *
 * head_stride + d, in elements.  Its type is bf16, fp16 or e4m3; an e4m3
 * cache has a power-of-two scale for each block and head, an e8m0 byte e at
 * scales + b * scale_block_stride + h * scale_head_stride for K and one
 * scale_side_stride further for V: a stored value v stands for v *
 * 2^(e - 127) (e = 255: NaN).
 *
 * Sequences: row s of the int32 block_tables ([n_seqs, table_width], rows
 * table_stride apart) names the blocks of sequence s in order, and the int32
 * lengths[s] its tokens, those of this step included.  Token rows of the
 * step's tensors are the sequences' last tokens: row query_starts[s] + i is
 * token lengths[s] - (query_starts[s + 1] - query_starts[s]) + i of sequence
 * s (query_starts: n_seqs + 1 int32, rising from 0); without query_starts
 * every sequence has one row, row s.  Rows past the last sequence's are
 * padding: they may be read, but nothing is written for them.  These tables are
 * read on the device and may change between replays of a captured launch.  A
 * table entry outside [0, blocks) names no block: nothing is written for it
 * and its tokens are seen by nobody; so are tokens past the table's width.
 * A length counts up to 2^30, and a table names fewer tokens than that.
 */
#ifndef KVSNAP_ATTENTION_H
#define KVSNAP_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { KVSNAP_BF16 = 0, KVSNAP_FP16 = 1, KVSNAP_E4M3 = 2, KVSNAP_FP32 = 3 };

typedef struct kvsnap_paged_layer {
    void* key;
    void* value;
    uint8_t* scales; /* NULL unless e4m3 */
    int64_t block_stride, token_stride, head_stride;
    int64_t scale_block_stride, scale_head_stride, scale_side_stride;
    int64_t blocks;
    int32_t block_size, kv_heads, width, type;
} kvsnap_paged_layer;

typedef struct kvsnap_sequences {
    const int32_t* block_tables;
    const int32_t* lengths;
    const int32_t* query_starts; /* or NULL */
    int64_t table_stride;
    int32_t table_width, n_seqs;
} kvsnap_sequences;

/* Positions and angles.  angles: fp32 [rows, pairs, 2], the cosine and sine
 * of pair j at each position (16-byte aligned); pairs is a multiple of 8.
 * Pair j turns values j and j + pairs of a head, or 2j and 2j + 1 where
 * `interleaved`; values from 2 * pairs on are left as they are.  positions:
 * int64 (or int32 where `narrow`), axis_stride apart for each axis; axes[u]
 * holds, two bits a pair from the lowest, the axis of pairs 8u..8u+7.
 * positions NULL: token i of a sequence is at i.  A position outside [0,
 * rows) has no angle: its turned values are NaN. */
typedef struct kvsnap_rotation {
    const float* angles; /* NULL: nothing is turned */
    const void* positions;
    int64_t rows, axis_stride;
    int32_t pairs, interleaved, narrow, inverse;
    uint16_t axes[16];
} kvsnap_rotation;

/* out = x with every head turned, for x and out of `tokens` rows of `heads`
 * heads of `width` values of type (bf16, fp16 or fp32), strides in elements;
 * `inverse` turns back, which is also the gradient's turn.  out may be x, and
 * otherwise overlaps no part of it.
 * width a multiple of 16 up to 256; rows, heads and angles 16-byte aligned. */
int kvsnap_rotate(const void* x, int64_t x_token_stride, int64_t x_head_stride, void* out, int64_t out_token_stride,
                  int64_t out_head_stride, int64_t tokens, int heads, int width, int type,
                  const kvsnap_rotation* rotation, uintptr_t stream);

/* One step's keys and values ([tokens, kv_heads, width] of type bf16 or fp16)
 * into their sequences' blocks, the keys turned on the way, and `query`
 * ([tokens, heads, width], or NULL) turned into query_out (which may be
 * query, and otherwise overlaps nothing that is read).  A 16-bit cache is of
 * the same type.  Into an e4m3 cache a block's values go with the least power
 * of two that keeps the new ones within e4m3's 448, or the block's scale where
 * slots filled before this step need more; where the new ones do, the slots
 * before them are rounded again to the new scale.  Slots past the sequence's
 * length are left as they are, and a value that is not finite is stored as
 * NaN.  No block that a call writes is named twice by the pages that it writes, of
 * one sequence or of several.  lengths[s] is at least the rows of sequence s;
 * rows ahead of position 0 are padding too. */
int kvsnap_append(const kvsnap_paged_layer* layer, const kvsnap_sequences* sequences, const kvsnap_rotation* rotation,
                  const void* key, int64_t key_token_stride, int64_t key_head_stride, const void* value,
                  int64_t value_token_stride, int64_t value_head_stride, const void* query, int64_t query_token_stride,
                  int64_t query_head_stride, void* query_out, int64_t out_token_stride, int64_t out_head_stride,
                  int64_t tokens, int heads, int type, uintptr_t stream);

/* Device bytes of scratch that kvsnap_attend needs over this layer (0: none);
 * ragged: whether it is given query_starts.  max_length: kvsnap_attend's, or
 * table_width * block_size if that is less. */
size_t kvsnap_attend_workspace_bytes(const kvsnap_paged_layer* layer, int64_t tokens, int n_seqs, int ragged, int heads,
                                     int64_t max_length, int64_t window);

/* out[row, h] = the sum over the tokens t that a row sees of softmax(scale *
 * query[row, h] . key[t]) value[t], for query and out of `tokens` rows of
 * `heads` heads (a multiple of the layer's, consecutive ones sharing a key
 * head) of type bf16 or fp16; a 16-bit cache is of the same type, and out may
 * be query, but otherwise overlaps no part of it.  The row at position p of its
 * sequence sees tokens 0..p, with window > 0 the last `window` of them; one
 * that sees none, or scores of -inf alone, has zeros and a log sum of -inf.
 * Softmax, sums and products' sums are fp32; weights are rounded to 16 bits
 * before they meet the values (to two such terms for fp16 queries over an
 * e4m3 cache; over an fp16 cache what is under 2^-30 of the largest among 64
 * tokens may vanish, which moves an output by at most 2^-24 of the largest
 * value), and an e4m3 cache's values are exact in bf16 at scales from 2^-117 to
 * 2^119 (past them, what is under 2^-126 may vanish and what is over bf16's largest
 * is infinite).  lse, or NULL:
 * fp32 [tokens, heads], the natural logarithm of each row's sum of
 * exponentials.  max_length, at least every sequence's length if it can be
 * known, only shapes the launch.  workspace: 16-byte aligned scratch of
 * kvsnap_attend_workspace_bytes bytes, used until the launch ends. */
int kvsnap_attend(const kvsnap_paged_layer* layer, const kvsnap_sequences* sequences, const void* query,
                  int64_t query_token_stride, int64_t query_head_stride, void* out, int64_t out_token_stride,
                  int64_t out_head_stride, float* lse, int64_t tokens, int heads, int type, float scale,
                  int64_t window, int64_t max_length, void* workspace, size_t workspace_bytes, uintptr_t stream);

#ifdef __cplusplus
}
#endif

#endif /* KVSNAP_ATTENTION_H */
