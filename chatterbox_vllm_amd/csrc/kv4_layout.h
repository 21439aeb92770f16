// Where the bytes of the 4-bit KV cache are.  Plain C++ without HIP types, so that host programs can check it.
//
// pool[layer][page][kv head][slab]; a page is 64 tokens of one stream, a slab 64 * (hd + hd / 16) bytes:
//   K codes | V codes | K scales [hd/32][64 tokens] | V scales [hd/32][64 tokens]
// A value is a 4-bit code (e2m1: 0, .5, 1, 1.5, 2, 3, 4, 6, sign in bit 3) times 2^(scale byte - 127); 32 consecutive dims of
// one (token, head) share a scale.  Byte 255 in the K scales marks an entry that stood for a NaN or an infinity.
//
// The codes are ordered as v_mfma_f32_16x16x32_bf16 takes them, one 16-byte load per lane (lane = 16 g + r) and 1 KiB of
// consecutive memory per wave:
//   K  A operand of S^T = K Q^T.  Row r of tile i is token 4 r + i; lane group g holds dims [g hd/4, (g+1) hd/4).  At hd 128 a
//      lane's 16 bytes are those 32 dims of one token, at hd 64 the 16 dims of two tokens (i, i + 1).
//   V  A operand of O^T = V^T P^T.  Row r of tile e is dim 64 h + 4 r + e; lane group g holds tokens 16 g + 8 s .. + 7, which is
//      where that product's B operand has them: the lane that computed S^T for 16 consecutive tokens and one query feeds P
//      back from its own registers.  A lane's 16 bytes are 4 dims (2 bytes) of 8 tokens.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define KV4_FN __host__ __device__ __forceinline__
#else
#define KV4_FN inline
#endif

#define KV4_PAGE 64
#define KV4_BLOCK 32             // dims that share a scale
#define KV4_NAN_SCALE 255        // K scale byte of an entry that held a non-finite value
#define KV4_MIN_SCALE 2          // smallest scale byte append writes: half a step, 2^(2 - 127) / 2, is the smallest normal float
#define KV4_MAX_SCALE 252        // largest: 6 * 2^(252 - 127) is finite in bf16

KV4_FN int kv4_slab_bytes(int hd) { return KV4_PAGE * (hd + hd / 16); }
// byte of the code of token t (0..63), dim d; the low nibble is the even dim
KV4_FN int kv4_k_at(int hd, unsigned t, unsigned d) {
    const unsigned q = hd / 4, two = 128 / hd;                       // dims per lane group; tokens per 16 bytes
    return (t % 4 / two) * 1024 + ((d / q) * 16 + t / 4) * 16 + (t % 4 % two) * 8 + d % q / 2;
}
KV4_FN int kv4_v_at(int hd, unsigned t, unsigned d) {
    return 32 * hd + (d / 64 * 2 + t / 8 % 2) * 1024 + ((t / 16) * 16 + d % 64 / 4) * 16 + t % 8 * 2 + d % 4 / 2;
}
KV4_FN int kv4_ks_at(int hd, unsigned t, unsigned d) { return 64 * hd + d / KV4_BLOCK * KV4_PAGE + t; }
KV4_FN int kv4_vs_at(int hd, unsigned t, unsigned d) { return 66 * hd + d / KV4_BLOCK * KV4_PAGE + t; }

// The batch of a call: sequence i owns rows [start, start + n) of the row tensors; they are entries ctx - n .. ctx - 1 of
// `stream`.  state: 0 = in order, 1 = to be skipped (stream < 0, or no rows), 2 = refused: numbers that do not fit the cache or
// the call.  Rows [start, start + n) always lie inside [0, rows), whatever the numbers on the device say.
struct Kv4Seq { int start, n, ctx, stream, state; };
KV4_FN Kv4Seq kv4_seq(int a, int b, int stream, int ctx, int rows, int max_rows, int n_streams, int64_t most) {
    Kv4Seq s;
    const int lo = a < 0 ? 0 : a < rows ? a : rows, hi = b < lo ? lo : b < rows ? b : rows;
    s.start = lo; s.n = hi - lo; s.ctx = ctx; s.stream = stream;
    s.state = (stream < 0 || s.n == 0) ? 1 : (a != lo || b != hi || s.n > max_rows || stream >= n_streams || ctx < 0 || ctx > most) ? 2 : 0;
    return s;
}
// page ids outside the pool are never followed
KV4_FN bool kv4_page_ok(int page, int n_pages) { return page >= 0 && page < n_pages; }
// scale byte of a block from the bits of its largest magnitude: the smallest power of two that leaves it below 7, which still
// rounds to the largest code, 6 (adding a quarter of the significand's range carries into the exponent from 1.75 on)
KV4_FN int kv4_scale_byte(unsigned amax_bits) {
    const int b = (int)((amax_bits + 0x200000u) >> 23) - 2;
    return b < KV4_MIN_SCALE ? KV4_MIN_SCALE : b > KV4_MAX_SCALE ? KV4_MAX_SCALE : b;
}
// order-preserving bits of an accumulated weight: larger weight, larger key; NaN counts as the lowest, -0 as 0
KV4_FN unsigned kv4_weight_key(unsigned bits) {
    if ((bits & 0x7fffffffu) > 0x7f800000u) return 0u;
    if (bits == 0x80000000u) bits = 0u;
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
