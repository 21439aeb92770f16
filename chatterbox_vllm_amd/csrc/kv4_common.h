// Device and host helpers shared by the kernels of the 4-bit KV cache (gfx950 only).
#pragma once
#include "t3_common.h"
#include "kv4_layout.h"
#include "../../include/t3_hip.h"

typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

struct Kv4View {                 // one layer of the cache
    uint8_t* pool;
    const int32_t* table;
    int n_pages, n_streams, max_pages, Hkv;
};
struct Kv4Rows {                 // the batch
    const int32_t* seq_start; const int32_t* stream; const int32_t* ctx;
    int n_seqs, rows, max_rows, max_ctx;
};

__device__ __forceinline__ Kv4Seq kv4_seq_of(const Kv4Rows& b, const Kv4View& c, int i) {
    const int64_t cap = (int64_t)c.max_pages * KV4_PAGE;
    return kv4_seq(b.seq_start[i], b.seq_start[i + 1], b.stream[i], b.ctx[i], b.rows, b.max_rows, c.n_streams, b.max_ctx < cap ? b.max_ctx : cap);
}
// 2^(byte - 127); 255 gives infinity, which the conversions below take for the scale's NaN
__device__ __forceinline__ float kv4_scale(unsigned byte) { return __uint_as_float(byte << 23); }
// byte `sel` of a word of codes times the scale: two values, exact in bf16 (an e2m1 value has two significant bits)
template <int SEL> __device__ __forceinline__ unsigned kv4_pair(unsigned codes, float scale) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL));
}

// ---- host side --------------------------------------------------------------------------------------------------------
int kv4_check_cache(const t3_kv4_cache* c, int layer, int n_layers, hipStream_t st);
int kv4_check_batch(const t3_kv4_batch* b);
inline Kv4View kv4_view(const t3_kv4_cache* c, int layer) {
    return Kv4View{static_cast<uint8_t*>(c->pool_dev) + (int64_t)layer * c->layer_stride, c->block_table_dev, c->n_pages, c->n_streams,
                   c->max_pages, c->Hkv};
}
inline Kv4Rows kv4_rows(const t3_kv4_batch* b) {
    return Kv4Rows{b->seq_start_dev, b->stream_dev, b->ctx_dev, b->n_seqs, b->rows, b->max_rows, b->max_ctx};
}
