// The 8-bit cache's kernels that other files' entry points launch.
#pragma once

#include <cstdint>

namespace wt {

// S new tokens per row over the row's cached slots and, causally, each other (kv8_prompt.cu).
int kv8_self_prompt(int dtype, const void *qkv, const void *k8, const void *v8, const float *ks, const float *vs,
                  const int64_t *offset, const int32_t *src, void *y, int rows, int new_tokens, int heads,
                  int capacity, void *stream);
// S queries per window over the window's frames, for more queries than a decode step has (kv8_tile.cu).
constexpr int kTileQueries = 128;
inline long long kv8_cross_tiles(int queries) { return (static_cast<long long>(queries) + kTileQueries - 1) / kTileQueries; }
int kv8_cross_tile(int dtype, const void *q, const void *k8, const void *v8, const float *ks, const float *vs,
                   const int64_t *lengths, void *y, int windows, int queries, int heads, int frames, int sms,
                   int *err, void *stream);
// The new tokens' keys and values into the cache at offset, offset + 1, ... (kv8_cache.cu); 2 rows heads new_tokens < 2^31.
int kv8_append(int dtype, const void *qkv, const int64_t *offset, void *k8, void *v8, float *ks, float *vs, int rows,
               int new_tokens, int heads, int capacity, void *stream);

}  // namespace wt
