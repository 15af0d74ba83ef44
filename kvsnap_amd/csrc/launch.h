// What the launchers of both kernel files share: a C entry point's errors.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/kvsnap_attention.h"
#include "common.h"

#include <cstdint>
#include <exception>
#include <stdexcept>
#include <string>

namespace kvsnap {

// 0, or -1 with the message of what `f` threw in the thread's error slot: no exception leaves a C entry point.
template <typename F>
int guarded(F&& f) {
    try {
        f();
        return 0;
    } catch (const std::exception& e) {
        set_error(e.what());
        return -1;
    }
}

inline void check_launched(const char* what) {
    const hipError_t rc = hipGetLastError();
    if (rc != hipSuccess) throw std::runtime_error(std::string(what) + " launch: " + hipGetErrorString(rc));
}

inline void require(bool held, const char* why) {
    if (!held) throw std::runtime_error(why);
}

// What every operator over a layer's cache asks of it: 16-byte pieces, and offsets that fit 32 bits of 16 bytes.
inline void check_layer(const kvsnap_paged_layer& layer) {
    require(layer.type == KVSNAP_BF16 || layer.type == KVSNAP_FP16 || layer.type == KVSNAP_E4M3,
            "the cache must be bf16, fp16 or e4m3");
    require(layer.blocks > 0 && layer.block_size > 0 && layer.kv_heads > 0, "the cache must not be empty");
    require(layer.block_size <= (1 << 20) && layer.blocks < (int64_t(1) << 31), "the cache's blocks are too many or long");
    require(layer.width > 0 && layer.width % 16 == 0 && layer.width <= 256,
            "the cache's width must be a multiple of 16 up to 256");
    require(layer.key && layer.value, "the cache needs device pointers");
    const int64_t element = layer.type == KVSNAP_E4M3 ? 1 : 2;
    require(reinterpret_cast<uintptr_t>(layer.key) % 16 == 0 && reinterpret_cast<uintptr_t>(layer.value) % 16 == 0 &&
                layer.block_stride * element % 16 == 0 && layer.token_stride * element % 16 == 0 &&
                layer.head_stride * element % 16 == 0,
            "the cache's rows must be 16-byte aligned");
    // A block's start and its slots' places are added in 32 bits of 16 bytes, and 16 slots' places in 32 bits of bytes.
    constexpr int64_t most = int64_t(1) << 36;
    require(layer.block_stride >= 0 && layer.token_stride >= 0 && layer.head_stride >= 0 && layer.block_stride < most &&
                layer.token_stride < (int64_t(1) << 26) &&
                (layer.blocks * __int128(layer.block_stride) + layer.block_size * layer.token_stride) * element < most,
            "the cache's K or V must be under 64 GiB, its strides not negative and a token's below 2^26");
    require((layer.scales != nullptr) == (layer.type == KVSNAP_E4M3), "an e4m3 cache has scales, another none");
}

inline void check_sequences(const kvsnap_sequences& q, const kvsnap_paged_layer& layer) {
    require(q.n_seqs >= 0 && q.table_width >= 0 && q.table_stride >= 0, "negative table size");
    require(int64_t(q.table_width) * layer.block_size < (int64_t(1) << 30), "the tables name 2^30 tokens or more");
    require(q.n_seqs == 0 || (q.lengths && (q.table_width == 0 || q.block_tables)), "the tables must be device pointers");
}

}  // namespace kvsnap
