// Attention over the 4-bit KV cache (byte order: kv4_layout.h).
//
// A column is a (row, query head) pair; the group = H / Hkv query heads of a key head and the rows of a sequence share its keys,
// so column c of a sequence and key head is row c / group, head c % group, and 16 columns make one tile of
//   S^T[token][column] = K Q^T        K codes -> bf16 in registers (exact), Q held in registers for the whole pass
//   O^T[dim][column]   = V^T P^T      P as bf16 hi + lo parts, so the probabilities keep 16 significant bits (bf16 prompts: hi)
// on v_mfma_f32_16x16x32_bf16, a page of 64 tokens at a time.  A lane ends the first product with 16 consecutive tokens of one
// column, which is what the second takes from it: no exchange but the maximum over the four lane groups.
// fp16 queries enter as bf16 hi + lo (exact to 2^-16 of the value, fp16 has 11 bits), so one set of products serves both types.
//
//   p = exp2((s - m) c),  c = scale log2(e),  m the running maximum of the scores themselves, l the running sum:  one pass, fp32.
// m follows the maximum in jumps: it stays while p is at most 2^8 (which costs fp32 and bf16 nothing), so the sums are rarely rescaled.
// The difference is taken before the product: it is exact near the maximum, whose p is then at least 1 at any size of s, and the factors
// between pages and chunks, exp2((m - m') c), agree with it.  (One fma(s, c, -m c) would leave the maximum the rounding of m c, which from
// m c = 2^31 on is more than all of fp32's exponents.)
//
// Sequences of at most KV4_FEW_COLUMNS columns (decode steps, drafted tokens) are cut into chunks of their cache, a workgroup of
// four waves each; a second launch joins the chunks in order.  Longer ones (prompts) run whole: a wave keeps one or two column tiles and
// walks the cache.  Which form and how many chunks follow from the sequence alone, so a row's bits do not depend on the batch.
//
// Few columns are bound by the cache's bytes where there are many (16 x 32 heads on 8 key heads of 128, 9000..32749 entries: 386 MB in
// 77 us, 5.0 TB/s) and by latency where there are few (64 x 16 heads of 64, 120..1000 entries: 39 MB in 13.5 us; one stream 5 us).
// Many are bound by the instructions: matrix and vector instructions of a SIMD hardly run beside each other (measured: a 16x16x32
// product 17.4 clocks, an fma 2.5, an exp2 9.7, mixed ones six sevenths of the sum or more), so both count, and the products stand in
// blocks, each change from one kind to the other costing about 5 clocks.  2 x 4095 rows x 32 heads on 8 of 128: 346 GFLOP in 351 us, 0.99
// PFLOP/s (fp16 rows, whose queries and P are two bf16 parts each: 542 us).
#include "kv4_common.h"

#include <type_traits>

#define KV4_FEW_COLUMNS 64        // rows x group up to which a sequence is cut along its cache
#define KV4_SLACK 8.f             // the reference moves when a maximum passes it by 2^8
#define KV4_NONE -3.402823466e38f // running maximum before the first visible token (the lowest finite: no score lies below, no difference of two is NaN)
// 2^((s - m) c)
__device__ __forceinline__ float kv4_exp(float s, float m, float c) { return __builtin_amdgcn_exp2f((s - m) * c); }

// A chunk is 16 pages: the four waves of its workgroup take four each.  (8 waves: 64 x 16 heads of 64 over up to 1000 entries 13.2 -> 14.9 us,
// 16 x 32 heads of 128 over up to 32k 77 -> 107; 32 pages: one sequence of 4k 13.5 -> 18.5, the long ones 76; 8 pages: 10 and 79, one of
// 1k 6.6 -> 10, drafts of 40 columns 27.2 -> 28.1.)
#define KV4_FEW_WAVES 4
#define KV4_CHUNK_PAGES 16
KV4_FN int kv4_chunks(int ctx) { return (int)(((int64_t)ctx + KV4_CHUNK_PAGES * KV4_PAGE - 1) / (KV4_CHUNK_PAGES * KV4_PAGE)); }

// Where weights are wanted, the scores of a (sequence, key head) of few columns are kept if they are at most `room` values: KV4_KEEP (4 MiB),
// less where a call's would take more than KV4_KEEP_BYTES in all.
#define KV4_KEEP (1 << 20)
#define KV4_KEEP_BYTES (1ll << 29)
KV4_FN int64_t kv4_kept_width(int64_t ctx) { return (ctx + KV4_PAGE - 1) / KV4_PAGE * KV4_PAGE; }
KV4_FN bool kv4_kept(int cols, int ctx, int64_t room) { return cols <= KV4_FEW_COLUMNS && cols * kv4_kept_width(ctx) <= room; }

// Where a buffer by (sequence, key head) has its parts: by the number of the sequence, each part as large as there may be one, or by its
// rows, each part as large as they ask for.  The host takes what is less: few rows under loose bounds, or few sequences, some of them
// prompts.  Below 2^32 either way (65535 sequences of 64 columns, 1024 key heads; scores are fewer).
struct Kv4Place {
    unsigned seq, head, row, row_head;
    __device__ __forceinline__ unsigned at(int i, int h, const Kv4Seq& s) const { return i * seq + h * head + s.start * row + h * s.n * row_head; }
};
struct Kv4Attn {
    const uint16_t* q; uint16_t* out;
    unsigned q_stride, out_stride, inv;        // row strides in elements; ceil(2^32 / group), 0 for a group of one
    int group, tiles, chunks;     // query heads per key head; column tiles and chunks that a sequence of few columns has at most
    float c;                      // scale * log2(e)
    // of sequences of few columns, from kv4_states_at() on: O before its division by l [chunk][hd], m and l [chunk]
    float* states;
    f32x2* ml;
    Kv4Place few;
    // for the weights, or null.  Columns of a (sequence, key head) start at kv4_column(), tiles of 16 of them being whole:
    f32x2* norm;                  // m and 1 / l of each column, where scores are formed again
    uint8_t* frags;               // the queries of each tile as the product takes them: [hd / 32][64 lanes][16 bytes]
    int slots;                    // tiles of a key head that these have room for
    uint8_t* images;              // [sequence][key head][pages]: pages as bf16 fragments, K's then V's; or null
    int pages;
    float* scores;                // raw scores where kv4_kept(), from kv4_scores_at() on: [column][kv4_kept_width]; or null
    Kv4Place kept;
    int64_t kept_unit, room;
    // row of a column: col / group without a division (exact below 2^26, and there are at most 2^22 columns)
    __device__ __forceinline__ int row(int col) const { return inv ? (int)__umulhi((unsigned)col, inv) : col; }
    __device__ __forceinline__ const uint16_t* q_at(int row, int head_at) const { return q + (uint64_t)(unsigned)row * q_stride + head_at; }
    __device__ __forceinline__ uint16_t* out_at(int row, int head_at) const { return out + (uint64_t)(unsigned)row * out_stride + head_at; }
};
// chunk states of a column of a sequence of few columns, one behind the other
__device__ __forceinline__ int64_t kv4_states_at(const Kv4Attn& a, int h, int seq, const Kv4Seq& s, int col) {
    return (int64_t)(a.few.at(seq, h, s) + col) * a.chunks;
}
// scores of a sequence and key head
__device__ __forceinline__ float* kv4_scores_at(const Kv4Attn& a, int h, int seq, const Kv4Seq& s) { return a.scores + a.kept.at(seq, h, s) * a.kept_unit; }

// first column of a sequence and key head: sequences in order take disjoint tiles, for floor((a + b) / 16) + 1 >= floor(a / 16) +
// ceil(b / 16), and never one outside the buffer
__device__ __forceinline__ int64_t kv4_column(const Kv4Attn& a, int h, int seq, const Kv4Seq& s) {
    return ((int64_t)h * a.slots + (s.start * a.group >> 4) + seq) * 16;
}

// Pages that one workgroup alone looks at are fetched past the caches (16 x 32 heads over up to 32k entries 88 -> 77 us); those that
// several column tiles share are not (drafts of 40 columns 17.9 us, 18.7 so).
template <bool ONCE, typename T> __device__ __forceinline__ T kv4_read_once(const T* p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(p);
    else return *p;
}

template <int HD> struct Kv4Page {
    u32x4 k[HD / 32], v[HD / 32], vs[HD / 64];
    unsigned ks;
    unsigned bad_k, good_v;                                       // all ones or all zeros, the same in every lane
    template <bool ONCE> __device__ __forceinline__ void load_k(const uint8_t* slab, int lane) {
        const int g = lane >> 4, r = lane & 15;
#pragma unroll
        for (int x = 0; x < HD / 32; ++x) k[x] = kv4_read_once<ONCE>(reinterpret_cast<const u32x4*>(slab + x * 1024 + lane * 16));
        ks = kv4_read_once<ONCE>(reinterpret_cast<const unsigned*>(slab + 64 * HD + g * (HD / 4) / KV4_BLOCK * KV4_PAGE + 4 * r));
    }
    template <bool ONCE> __device__ __forceinline__ void load_v(const uint8_t* slab, int lane) {
        const int g = lane >> 4, r = lane & 15;
#pragma unroll
        for (int x = 0; x < HD / 32; ++x) v[x] = kv4_read_once<ONCE>(reinterpret_cast<const u32x4*>(slab + 32 * HD + x * 1024 + lane * 16));
#pragma unroll
        for (int x = 0; x < HD / 64; ++x) vs[x] = kv4_read_once<ONCE>(reinterpret_cast<const u32x4*>(slab + 66 * HD + (2 * x + (r >> 3)) * KV4_PAGE + 16 * g));
    }
};
__device__ __forceinline__ unsigned kv4_byte(unsigned w, int i) { return w >> (8 * i) & 255u; }

// Q of one column tile: step x of the product takes dims g hd/4 + 8 x .. + 7 of lane group g
template <int HD, bool F16> struct Kv4Query {
    bf16x8 q[(F16 ? 2 : 1) * HD / 32];
    __device__ __forceinline__ void set(int x, u32x4 w) {
        if constexpr (F16) {
            const f16x8 f = __builtin_bit_cast(f16x8, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const __bf16 hi = (__bf16)(float)f[e];
                q[x][e] = hi;
                q[HD / 32 + x][e] = (__bf16)((float)f[e] - (float)hi);
            }
        } else {
            q[x] = __builtin_bit_cast(bf16x8, w);
        }
    }
    // from a row (null: a column that is none), and, if wanted, on to where the weights' pass finds the tile
    __device__ __forceinline__ void load(const uint16_t* row, int lane, uint8_t* keep) {
#pragma unroll
        for (int x = 0; x < HD / 32; ++x) {
            u32x4 w = {0u, 0u, 0u, 0u};
            if (row) w = *reinterpret_cast<const u32x4*>(row + (lane >> 4) * (HD / 4) + 8 * x);
            if (keep) *reinterpret_cast<u32x4*>(keep + x * 1024 + lane * 16) = w;
            set(x, w);
        }
    }
};

// K of a page as operands of the first product: tile i, step x
template <int HD> __device__ __forceinline__ void kv4_operands(const Kv4Page<HD>& pg, bf16x8 (&kf)[4][HD / 32]) {
    const unsigned ks = pg.ks | pg.bad_k;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float sc = kv4_scale(kv4_byte(ks, i));
#pragma unroll
        for (int x = 0; x < HD / 32; ++x) {
            const unsigned w = HD == 64 ? pg.k[i / 2][i % 2 * 2 + x] : pg.k[HD == 64 ? 0 : i][x];
            const u32x4 a = {kv4_pair<0>(w, sc), kv4_pair<1>(w, sc), kv4_pair<2>(w, sc), kv4_pair<3>(w, sc)};
            kf[i][x] = __builtin_bit_cast(bf16x8, a);
        }
    }
}

// S^T of a page for NC column tiles: s[n][i][j] = token 16 g + 4 j + i, column lane & 15
template <int HD, bool F16, int NC>
__device__ __forceinline__ void kv4_scores(const Kv4Page<HD>& pg, const Kv4Query<HD, F16> (&q)[NC], f32x4 (&s)[NC][4]) {
    bf16x8 kf[4][HD / 32];
    kv4_operands<HD>(pg, kf);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int n = 0; n < NC; ++n) s[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < HD / 32; ++x)
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                s[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i][x], q[n].q[x], s[n][i], 0, 0, 0);
                if constexpr (F16) s[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i][x], q[n].q[HD / 32 + x], s[n][i], 0, 0, 0);
            }
    }
}

// running softmax state of NC column tiles.  m is the same in the four lanes of a column, l a lane's own share;
// o[n][h][e][j] = dim 64 h + 16 g + 4 j + e
template <int HD, int NC> struct Kv4State {
    float m[NC], l[NC];
    f32x4 o[NC][HD / 64][4];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            m[n] = KV4_NONE; l[n] = 0.f;
#pragma unroll
            for (int h = 0; h < HD / 64; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][h][e] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
};

// What a page that is not seen whole needs: scores of tokens behind a column's last one go to -inf (seen[n]: how many of the page
// it sees), and the value scales behind the last entry of the stream to 0, for those bytes may be anything and 0 * finite is 0.
template <int NC> __device__ __forceinline__ void kv4_hide_scores(f32x4 (&s)[NC][4], const int (&seen)[NC], int lane) {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int mine = seen[n] - 16 * (lane >> 4);              // of the lane's 16 tokens
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[n][i][j] = 4 * j + i < mine ? s[n][i][j] : -INFINITY;
    }
}
template <int HD> __device__ __forceinline__ void kv4_hide_values(Kv4Page<HD>& pg, int tail, int lane) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int mine = tail - 16 * (lane >> 4) - 4 * w;         // of the word's 4 tokens
        const unsigned keep = mine >= 4 ? 0xffffffffu : mine <= 0 ? 0u : (1u << (8 * mine)) - 1u;
#pragma unroll
        for (int x = 0; x < HD / 64; ++x) pg.vs[x][w] &= keep;
    }
}

// over the four lane groups
__device__ __forceinline__ float kv4_group_max(float x) {
    const unsigned u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned v = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float kv4_group_sum(float x) {
    const unsigned u = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned v = __float_as_uint(__uint_as_float(a[0]) + __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// over the 16 lanes of a group: neighbours, pairs, quads, eights (each step's operands are equal in the lanes that hold them)
template <int CTRL> __device__ __forceinline__ float kv4_lane_add(float x) {
    return x + __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float kv4_row_sum(float x) { return kv4_lane_add<0x140>(kv4_lane_add<0x141>(kv4_lane_add<0x4e>(kv4_lane_add<0xb1>(x)))); }
// two values as bf16 hi and lo parts, one word each
__device__ __forceinline__ void kv4_split(float p0, float p1, unsigned& hi, unsigned& lo) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    hi = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{p0, p1}), bf16x2));
    lo = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2{p0 - bf_lo(hi), p1 - bf_hi(hi)}), bf16x2));
}

// A page's softmax in two parts.  First the reference: it moves, and the sums with it, where a maximum has left it behind.
template <int HD, int NC> __device__ __forceinline__ void kv4_reference(const f32x4 (&s)[NC][4], Kv4State<HD, NC>& st, float c) {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        float top = s[n][0][0];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) top = fmaxf(top, s[n][i][j]);
        top = kv4_group_max(top);
        const float m = (top - st.m[n]) * c > KV4_SLACK ? top : st.m[n];
        if (__any(m != st.m[n])) {                                // a column that keeps its reference multiplies by one
            const float alpha = kv4_exp(st.m[n], m, c);
            st.m[n] = m;
            st.l[n] *= alpha;
#pragma unroll
            for (int h = 0; h < HD / 64; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) st.o[n][h][e] *= alpha;
        }
    }
}
// Then the probabilities.  ph + pl: slot y of step x is token 16 g + 8 x + y; without LO, ph alone.
template <int HD, int NC, bool LO>
__device__ __forceinline__ void kv4_probabilities(const f32x4 (&s)[NC][4], Kv4State<HD, NC>& st, float c, bf16x8 (&ph)[NC][2], bf16x8 (&pl)[NC][2]) {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        float sum = 0.f;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            u32x4 hi, lo;
#pragma unroll
            for (int y = 0; y < 8; y += 2) {
                const int e = 8 * x + y;                          // tokens 16 g + e, + e + 1
                const float p0 = kv4_exp(s[n][e & 3][e >> 2], st.m[n], c);
                const float p1 = kv4_exp(s[n][(e & 3) + 1][e >> 2], st.m[n], c);
                sum += p0 + p1;
                unsigned h, l;
                kv4_split(p0, p1, h, l);
                hi[y / 2] = h; lo[y / 2] = l;
            }
            ph[n][x] = __builtin_bit_cast(bf16x8, hi);
            if constexpr (LO) pl[n][x] = __builtin_bit_cast(bf16x8, lo);
        }
        st.l[n] += sum;
    }
}

// O^T += V^T P^T of one page
template <int HD, int NC>
__device__ __forceinline__ void kv4_values(const Kv4Page<HD>& pg, const bf16x8 (&ph)[NC][2], const bf16x8 (&pl)[NC][2], Kv4State<HD, NC>& st) {
#pragma unroll
    for (int h = 0; h < HD / 64; ++h)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            u32x4 a[4];                                           // tile e: 8 tokens of dim 64 h + 4 r + e
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const unsigned codes = pg.v[2 * h + x][w];
                const int t = 8 * x + 2 * w;                      // tokens 16 g + t, + t + 1
                const unsigned vs = pg.vs[h][t / 4] & pg.good_v;
                const float s0 = kv4_scale(kv4_byte(vs, t % 4)), s1 = kv4_scale(kv4_byte(vs, t % 4 + 1));
                const unsigned t0 = kv4_pair<0>(codes, s0), t0b = kv4_pair<1>(codes, s0);
                const unsigned t1 = kv4_pair<2>(codes, s1), t1b = kv4_pair<3>(codes, s1);
                a[0][w] = __builtin_amdgcn_perm(t1, t0, 0x05040100u);
                a[1][w] = __builtin_amdgcn_perm(t1, t0, 0x07060302u);
                a[2][w] = __builtin_amdgcn_perm(t1b, t0b, 0x05040100u);
                a[3][w] = __builtin_amdgcn_perm(t1b, t0b, 0x07060302u);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bf16x8 af = __builtin_bit_cast(bf16x8, a[e]);
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    st.o[n][h][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, ph[n][x], st.o[n][h][e], 0, 0, 0);
                    st.o[n][h][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, pl[n][x], st.o[n][h][e], 0, 0, 0);
                }
            }
        }
}

// Two outputs.  In fp16 cut at the type's largest, as read cuts them: an entry appended from fp16 can be held as up to 65536.  (The bits of
// an infinity less one are those of the largest; a NaN stays one.)
template <bool F16> __device__ __forceinline__ unsigned kv4_pack2(float lo, float hi) {
    if constexpr (F16) {
        typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
        const f16x2 p = {(_Float16)lo, (_Float16)hi};
        u16x2 u = __builtin_bit_cast(u16x2, p);
        u -= (u & (uint16_t)0x7fff) == (uint16_t)0x7c00 ? u16x2{1, 1} : u16x2{0, 0};
        return __builtin_bit_cast(unsigned, u);
    } else {
        return pack_bf2(lo, hi);
    }
}
// A page of a stream.  An id outside the pool is not followed: the page then holds NaN keys, and values that a row which does not
// see it can multiply by zero.  `bad` is applied where the bytes are used, so that nothing waits for a load when it is issued.
template <int HD> __device__ __forceinline__ const uint8_t* kv4_slab_of(const Kv4View& c, int page, int h) {
    return c.pool + ((int64_t)(kv4_page_ok(page, c.n_pages) ? page : 0) * c.Hkv + h) * kv4_slab_bytes(HD);
}
template <int HD, bool ONCE> __device__ __forceinline__ void kv4_fetch_k(Kv4Page<HD>& pg, const Kv4View& c, int page, int h, int lane) {
    pg.bad_k = kv4_page_ok(page, c.n_pages) ? 0u : 0xffffffffu;
    pg.template load_k<ONCE>(kv4_slab_of<HD>(c, page, h), lane);
}
template <int HD, bool ONCE> __device__ __forceinline__ void kv4_fetch_v(Kv4Page<HD>& pg, const Kv4View& c, int page, int h, int lane) {
    pg.good_v = kv4_page_ok(page, c.n_pages) ? 0xffffffffu : 0u;
    pg.template load_v<ONCE>(kv4_slab_of<HD>(c, page, h), lane);
}
// bits of a NaN in both halves of a word, of either type
#define KV4_NAN2 0x7fff7fffu

// NaN into the rows of columns [c0, c1) of a sequence and key head
template <int HD> __device__ void kv4_fill_columns(const Kv4Attn& a, const Kv4Seq& s, int h, int c0, int c1, int tid, int threads) {
    for (int i = tid; i < (c1 - c0) * (HD / 8); i += threads) {
        const int col = c0 + i / (HD / 8), j = a.row(col), head = h * a.group + col - j * a.group;
        const u32x4 w = {KV4_NAN2, KV4_NAN2, KV4_NAN2, KV4_NAN2};
        *reinterpret_cast<u32x4*>(a.out_at(s.start + j, head * HD + i % (HD / 8) * 8)) = w;
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Few columns: one workgroup per (chunk, tile of 16 columns and key head, sequence).
// ------------------------------------------------------------------------------------------------------------------
template <int HD> struct Kv4FewLds {
    float m[KV4_FEW_WAVES][2][16];
    __attribute__((aligned(16))) float o[KV4_FEW_WAVES][16][HD + 4];
};

template <int HD, bool F16, bool ONCE>
__device__ __forceinline__ void kv4_few_block(const Kv4View& c, const Kv4Rows& b, const Kv4Attn& a, Kv4FewLds<HD>& lds, int h, int tile, int seq, int chunk) {
    float (&sm)[KV4_FEW_WAVES][2][16] = lds.m;
    float (&so)[KV4_FEW_WAVES][16][HD + 4] = lds.o;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Kv4Seq s = kv4_seq_of(b, c, seq);
    const int rows = s.n < b.max_rows ? s.n : b.max_rows;
    const int cols = rows * a.group;
    if (s.state == 1 || cols > KV4_FEW_COLUMNS || tile * 16 >= cols) return;
    const int c1 = cols < tile * 16 + 16 ? cols : tile * 16 + 16;
    if (s.state == 2) {
        if (chunk == 0) kv4_fill_columns<HD>(a, s, h, tile * 16, c1, tid, 64 * KV4_FEW_WAVES);
        return;
    }
    const int chunks = kv4_chunks(s.ctx);
    if (chunk >= (chunks > 0 ? chunks : 1)) return;

    const int col = tile * 16 + (lane & 15), j = a.row(col), head = h * a.group + col - j * a.group;
    const int sees = col < cols ? s.ctx - s.n + j + 1 : 0;        // entries that this lane's column sees, may be <= 0
    const int least = s.ctx - s.n + a.row(tile * 16) + 1;    // what the tile's first row sees
    Kv4Query<HD, F16> q[1];
    q[0].load(col < cols ? a.q_at(s.start + j, head * HD) : nullptr, lane,
              a.frags && !kv4_kept(cols, s.ctx, a.room) && chunk == 0 && w == 0 ? a.frags + (kv4_column(a, h, seq, s) + tile * 16) * (2 * HD) : nullptr);
    Kv4State<HD, 1> st;
    st.clear();

    const int p0 = chunk * KV4_CHUNK_PAGES, pages = (s.ctx + KV4_PAGE - 1) / KV4_PAGE;
    const int np = pages - p0 < KV4_CHUNK_PAGES ? pages - p0 : KV4_CHUNK_PAGES;
    // the chunk's page ids, one a lane.  The next page's keys are under way from when this one's have been used, its values
    // likewise: half a step of other work covers each load, in the registers of one page
    const int32_t* bt = c.table + (int64_t)s.stream * c.max_pages + p0;
    const int ids = lane < np ? bt[lane] : -1;
    // where the lane's 16 tokens' scores go, if they are wanted
    float* keep = a.scores && col < cols && kv4_kept(cols, s.ctx, a.room)
                      ? kv4_scores_at(a, h, seq, s) + col * kv4_kept_width(s.ctx) + 16 * (lane >> 4) : nullptr;
    Kv4Page<HD> pg;
    if (w < np) {
        const int id = __builtin_amdgcn_readlane(ids, w);
        kv4_fetch_k<HD, ONCE>(pg, c, id, h, lane);
        kv4_fetch_v<HD, ONCE>(pg, c, id, h, lane);
    }
    // (the last page has a body of its own: a load under a condition would make every wait below one for all loads)
    const auto step = [&](int p, auto more) {
        const int first = (p0 + p) * KV4_PAGE, seen[1] = {sees - first};
        const int next = more() ? __builtin_amdgcn_readlane(ids, p + KV4_FEW_WAVES) : 0;
        f32x4 sc[1][4];
        bf16x8 ph[1][2], pl[1][2];
        kv4_scores<HD, F16, 1>(pg, q, sc);
        if (keep) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
                *reinterpret_cast<f32x4*>(keep + first + 4 * x) = f32x4{sc[0][0][x], sc[0][1][x], sc[0][2][x], sc[0][3][x]};
        }
        if constexpr (more()) kv4_fetch_k<HD, ONCE>(pg, c, next, h, lane);
        if (least < first + KV4_PAGE) {
            kv4_hide_scores<1>(sc, seen, lane);
            kv4_hide_values<HD>(pg, s.ctx - first, lane);
        }
        kv4_reference<HD, 1>(sc, st, a.c);
        kv4_probabilities<HD, 1, true>(sc, st, a.c, ph, pl);
        kv4_values<HD, 1>(pg, ph, pl, st);
        if constexpr (more()) kv4_fetch_v<HD, ONCE>(pg, c, next, h, lane);
    };
    int p = w;
    for (; p + KV4_FEW_WAVES < np; p += KV4_FEW_WAVES) step(p, std::true_type{});
    if (p < np) step(p, std::false_type{});
    float l = st.l[0];
    l = kv4_group_sum(l);
    const int g = lane >> 4, cc = lane & 15;
    if (g == 0) { sm[w][0][cc] = st.m[0]; sm[w][1][cc] = l; }
#pragma unroll
    for (int x = 0; x < HD / 64; ++x)
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
            const f32x4 v = {st.o[0][x][0][jj], st.o[0][x][1][jj], st.o[0][x][2][jj], st.o[0][x][3][jj]};
            *reinterpret_cast<f32x4*>(&so[w][cc][64 * x + 16 * g + 4 * jj]) = v;
        }
    __syncthreads();
    // the waves in order; a thread 8 dims of a column
    for (int i = tid; i < 16 * (HD / 8); i += 64 * KV4_FEW_WAVES) {
        const int k = i / (HD / 8), d = i % (HD / 8) * 8, kcol = tile * 16 + k;
        if (kcol >= c1) continue;
        float M = sm[0][0][k];
#pragma unroll
        for (int x = 1; x < KV4_FEW_WAVES; ++x) M = fmaxf(M, sm[x][0][k]);
        float L = 0.f, o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = 0.f;
#pragma unroll
        for (int x = 0; x < KV4_FEW_WAVES; ++x) {
            const float f = kv4_exp(sm[x][0][k], M, a.c);
            L = fmaf(sm[x][1][k], f, L);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = fmaf(so[x][k][d + e], f, o[e]);
        }
        const int64_t at = kv4_states_at(a, h, seq, s, kcol) + chunk;
        if (a.ml && d == 0) a.ml[at] = f32x2{M, L};
        if (chunks > 1) {
            float* sp = a.states + at * HD + d;
#pragma unroll
            for (int e = 0; e < 8; e += 4) *reinterpret_cast<f32x4*>(sp + e) = f32x4{o[e], o[e + 1], o[e + 2], o[e + 3]};
        } else {
            const int jj = a.row(kcol), hh = h * a.group + kcol - jj * a.group;
            const float inv = L == 0.f ? 0.f : 1.0f / L;          // nothing seen: 0 (a NaN stays one)
            const u32x4 r = {kv4_pack2<F16>(o[0] * inv, o[1] * inv), kv4_pack2<F16>(o[2] * inv, o[3] * inv),
                             kv4_pack2<F16>(o[4] * inv, o[5] * inv), kv4_pack2<F16>(o[6] * inv, o[7] * inv)};
            *reinterpret_cast<u32x4*>(a.out_at(s.start + jj, hh * HD + d)) = r;
            if (a.norm && d == 0) a.norm[kv4_column(a, h, seq, s) + kcol] = f32x2{M, inv};
        }
    }
}

template <int HD, bool F16, bool ONCE>
__global__ __launch_bounds__(64 * KV4_FEW_WAVES, HD == 64 ? 4 : 2) void kv4_attn_few_kernel(Kv4View c, Kv4Rows b, Kv4Attn a) {
    __shared__ Kv4FewLds<HD> lds;
    kv4_few_block<HD, F16, ONCE>(c, b, a, lds, blockIdx.x % c.Hkv, blockIdx.x / c.Hkv, blockIdx.y, blockIdx.z);
}

// Joins the chunks of a column.  A thread has 4 dims; 1024 / HD groups of threads walk the chunks side by side, group x the chunks
// x, x + groups, ..., and are then added in order.  Latency: 4 to 5 us at 64 x 16 heads x 2 chunks and at 16 x 32 heads x 32 chunks.
template <int HD> struct Kv4JoinLds {
    f32x2 ml[1024 / HD];
    f32x4 o[1024 / HD][HD / 4];
};
template <int HD, bool F16>
__device__ __forceinline__ void kv4_join_block(const Kv4View& c, const Kv4Rows& b, const Kv4Attn& a, Kv4JoinLds<HD>& lds, int h, int col, int seq) {
    constexpr int T = HD / 4, GROUPS = 256 / T;
    const Kv4Seq s = kv4_seq_of(b, c, seq);
    const int rows = s.n < b.max_rows ? s.n : b.max_rows, cols = rows * a.group;
    if (s.state || cols > KV4_FEW_COLUMNS || col >= cols) return;
    const int chunks = kv4_chunks(s.ctx);
    if (chunks <= 1) return;
    const int group = threadIdx.x / T, t = threadIdx.x % T;
    const int64_t at = kv4_states_at(a, h, seq, s, col);
    const f32x2* ml = a.ml + at;
    const float* sp = a.states + at * HD + 4 * t;
    float M = KV4_NONE, L = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int x = group; x < chunks; x += GROUPS) {
        const f32x2 part = ml[x];
        const f32x4 v = *reinterpret_cast<const f32x4*>(sp + (int64_t)x * HD);
        const float top = fmaxf(M, part[0]), f0 = kv4_exp(M, top, a.c), f1 = kv4_exp(part[0], top, a.c);
        L = fmaf(L, f0, part[1] * f1);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(o[e], f0, v[e] * f1);
        M = top;
    }
    if (t == 0) lds.ml[group] = f32x2{M, L};
    lds.o[group][t] = o;
    __syncthreads();
    if (threadIdx.x >= T) return;
    M = lds.ml[0][0];
#pragma unroll
    for (int x = 1; x < GROUPS; ++x) M = fmaxf(M, lds.ml[x][0]);
    L = 0.f;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int x = 0; x < GROUPS; ++x) {
        const float f = kv4_exp(lds.ml[x][0], M, a.c);
        L = fmaf(lds.ml[x][1], f, L);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(lds.o[x][t][e], f, o[e]);
    }
    const int j = a.row(col), head = h * a.group + col - j * a.group;
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    const u32x2 r = {kv4_pack2<F16>(o[0] * inv, o[1] * inv), kv4_pack2<F16>(o[2] * inv, o[3] * inv)};
    *reinterpret_cast<u32x2*>(a.out_at(s.start + j, head * HD + 4 * t)) = r;
    if (a.norm && t == 0) a.norm[kv4_column(a, h, seq, s) + col] = f32x2{M, inv};
}
template <int HD, bool F16>
__global__ __launch_bounds__(256) void kv4_attn_join_kernel(Kv4View c, Kv4Rows b, Kv4Attn a) {
    __shared__ __attribute__((aligned(16))) Kv4JoinLds<HD> lds;
    const int col = blockIdx.x / c.Hkv;
    kv4_join_block<HD, F16>(c, b, a, lds, blockIdx.x - col * c.Hkv, col, blockIdx.y);
}

// ------------------------------------------------------------------------------------------------------------------
// Many columns (prompts): a workgroup of four waves takes 4 x NC tiles of 16 columns of a key head and walks the cache up to what
// its last row sees.  Each page is turned into bf16 once per workgroup: a wave converts a quarter (one of K's four token tiles, a
// quarter of V) and leaves it in LDS in operand order, 1 KiB per fragment and a lane's 16 bytes where the same lane of every
// wave will read them, while the products of the page before run from the other half of the buffer: one barrier a page.
// For bf16 rows P is rounded to bf16: each probability is off by at most 2^-8 of itself, independently, which adds an error of the
// size of the output's own rounding (at most 1.42 times it in all, measured over flat to sharp scores) and halves the second
// product (2 x 4095 rows x 32 heads of 128: 386 us against 476 with hi + lo parts, pages converted by each workgroup).  For fp16 rows P is hi + lo.
// ------------------------------------------------------------------------------------------------------------------
template <int HD> struct Kv4Stage {
    u32x4 k, v;                                                   // at hd 64 a wave's part of K is 8 bytes
    u32x2 vs;
    unsigned ks, bad_k, good_v;
    // wave w: token tile w of K; V at hd 128 the half (h, x) = (w / 2, w % 2), at hd 64 x = w / 2 and two of its four dim tiles
    __device__ __forceinline__ void load_k(const Kv4View& c, int page, int h, int w, int lane) {
        const int g = lane >> 4, r = lane & 15;
        bad_k = kv4_page_ok(page, c.n_pages) ? 0u : 0xffffffffu;
        const uint8_t* slab = kv4_slab_of<HD>(c, page, h);
        if constexpr (HD == 64) {
            const u32x2 t = *reinterpret_cast<const u32x2*>(slab + (w >> 1) * 1024 + lane * 16 + (w & 1) * 8);
            k = u32x4{t[0], t[1], 0u, 0u};
        } else {
            k = *reinterpret_cast<const u32x4*>(slab + w * 1024 + lane * 16);
        }
        ks = slab[64 * HD + g * (HD / 4) / KV4_BLOCK * KV4_PAGE + 4 * r + w];
    }
    __device__ __forceinline__ void load_v(const Kv4View& c, int page, int h, int w, int lane) {
        const int g = lane >> 4, r = lane & 15;
        good_v = kv4_page_ok(page, c.n_pages) ? 0xffffffffu : 0u;
        const uint8_t* slab = kv4_slab_of<HD>(c, page, h);
        const int part = HD == 64 ? w >> 1 : w;
        v = *reinterpret_cast<const u32x4*>(slab + 32 * HD + part * 1024 + lane * 16);
        vs = *reinterpret_cast<const u32x2*>(slab + 66 * HD + (HD == 64 ? r >> 3 : 2 * (w >> 1) + (r >> 3)) * KV4_PAGE + 16 * g + 8 * (HD == 64 ? part : w & 1));
    }
    __device__ __forceinline__ void store_k(uint8_t* buf, int w, int lane) const {
        const float sc = kv4_scale((ks | bad_k) & 255u);
#pragma unroll
        for (int y = 0; y < HD / 32; ++y) {
            const u32x4 a = {kv4_pair<0>(k[y], sc), kv4_pair<1>(k[y], sc), kv4_pair<2>(k[y], sc), kv4_pair<3>(k[y], sc)};
            *reinterpret_cast<u32x4*>(buf + (w * (HD / 32) + y) * 1024 + lane * 16) = a;
        }
    }
    // tail: tokens of the page that exist; the scales of the others go to 0 (their bytes may be anything, and 0 * finite is 0)
    __device__ __forceinline__ void store_v(uint8_t* buf, int tail, int w, int lane) const {
        const int x = HD == 64 ? w >> 1 : w & 1;
        u32x2 s;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int mine = tail - 16 * (lane >> 4) - 8 * x - 4 * z;
            s[z] = vs[z] & good_v & (mine >= 4 ? 0xffffffffu : mine <= 0 ? 0u : (1u << (8 * mine)) - 1u);
        }
        u32x4 a[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) {
            const float s0 = kv4_scale(kv4_byte(s[z / 2], z % 2 * 2)), s1 = kv4_scale(kv4_byte(s[z / 2], z % 2 * 2 + 1));
            const unsigned codes = HD == 64 && (w & 1) ? v[z] >> 8 : v[z];      // hd 64: dims 2, 3 move to where 0, 1 are
            const unsigned t0 = kv4_pair<0>(codes, s0), t1 = kv4_pair<2>(codes, s1);
            a[0][z] = __builtin_amdgcn_perm(t1, t0, 0x05040100u);
            a[1][z] = __builtin_amdgcn_perm(t1, t0, 0x07060302u);
            if constexpr (HD == 128) {
                const unsigned u0 = kv4_pair<1>(codes, s0), u1 = kv4_pair<3>(codes, s1);
                a[2][z] = __builtin_amdgcn_perm(u1, u0, 0x05040100u);
                a[3][z] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
            }
        }
        // fragment (h, x, e) of V
        const int f = HD == 64 ? x * 4 + 2 * (w & 1) : w * 4;
#pragma unroll
        for (int e = 0; e < HD / 32; ++e) *reinterpret_cast<u32x4*>(buf + (f + e) * 1024 + lane * 16) = a[e];
    }
};

// The order wanted of a product's block: four fragments read ahead, and one more behind the products of each, so that no product
// waits for LDS.  Nothing else is put between them: on this chip vector instructions hardly run beside matrix ones, of the same or
// of another wave (17.4 clocks a product, 27.5 with four fmas behind each), and every change from one to the other costs ~5 clocks.
template <int FRAGMENTS, int PRODUCTS> __device__ __forceinline__ void kv4_interleave() {
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);           // LDS reads
#pragma unroll
    for (int f = 0; f < FRAGMENTS; ++f) {
        __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS, 0);
        if (f + 4 < FRAGMENTS) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
}

// Where many workgroups look at each page it is converted once for all of them: a launch before leaves the pages' fragments in memory as
// they stand in LDS, where loads without a register on the way bring them (2 x 4095 rows x 32 heads of 128: 36 us less of 384, the 10 us of
// the conversion counted; through registers 30).
template <int HD> __device__ __forceinline__ uint8_t* kv4_image(const Kv4Attn& a, int Hkv, int seq, int h, int p) {
    return a.images + (((int64_t)seq * Hkv + h) * a.pages + p) * (256 * HD);
}
// wave w's quarter: half of K's or of V's fragments, 1 KiB a load
template <int HD> __device__ __forceinline__ void kv4_image_to_lds(const uint8_t* from, uint8_t* k, uint8_t* v, int w, int lane) {
    uint8_t* to = (w < 2 ? k : v) + (w & 1) * (HD * 64);
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + (w * (HD / 16) + i) * 1024 + lane * 16),
                                         (__attribute__((address_space(3))) void*)(to + i * 1024), 16, 0, 0);
}
template <int HD>
__global__ __launch_bounds__(256) void kv4_image_kernel(Kv4View c, Kv4Rows b, Kv4Attn a) {
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), p = blockIdx.x / c.Hkv, h = blockIdx.x - p * c.Hkv;
    const Kv4Seq s = kv4_seq_of(b, c, blockIdx.y);
    const int rows = s.n < b.max_rows ? s.n : b.max_rows;
    if (s.state || rows * a.group <= KV4_FEW_COLUMNS || p * KV4_PAGE >= s.ctx) return;
    const int id = __builtin_amdgcn_readfirstlane(c.table[(int64_t)s.stream * c.max_pages + p]);
    uint8_t* to = kv4_image<HD>(a, c.Hkv, blockIdx.y, h, p);
    Kv4Stage<HD> stage;
    stage.load_k(c, id, h, w, lane);
    stage.load_v(c, id, h, w, lane);
    stage.store_k(to, w, lane);
    stage.store_v(to + 128 * HD, s.ctx - p * KV4_PAGE, w, lane);
}

// S^T of a page from its fragments in LDS
template <int HD, bool F16, int NC>
__device__ __forceinline__ void kv4_lds_scores(const uint8_t* kbuf, const Kv4Query<HD, F16> (&q)[NC], f32x4 (&s)[NC][4], int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < NC; ++n) s[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < HD / 32; ++x) {                           // tiles inside steps: products of one sum lie 4 x NC apart
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bf16x8 af = *reinterpret_cast<const bf16x8*>(kbuf + (i * (HD / 32) + x) * 1024 + lane * 16);
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                s[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, q[n].q[x], s[n][i], 0, 0, 0);
                if constexpr (F16) s[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, q[n].q[HD / 32 + x], s[n][i], 0, 0, 0);
            }
        }
    }
}
template <int HD, bool LO, int NC>
__device__ __forceinline__ void kv4_lds_values(const uint8_t* vbuf, const bf16x8 (&ph)[NC][2], const bf16x8 (&pl)[NC][2], Kv4State<HD, NC>& st, int lane) {
#pragma unroll
    for (int hh = 0; hh < HD / 64; ++hh)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bf16x8 af = *reinterpret_cast<const bf16x8*>(vbuf + ((hh * 2 + x) * 4 + e) * 1024 + lane * 16);
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    st.o[n][hh][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, ph[n][x], st.o[n][hh][e], 0, 0, 0);
                    if constexpr (LO) st.o[n][hh][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, pl[n][x], st.o[n][hh][e], 0, 0, 0);
                }
            }
}

template <int HD> struct Kv4ManyLds { __attribute__((aligned(16))) uint8_t k[2][128 * HD], v[2][128 * HD]; };

template <int HD, bool F16, int NC, bool IMAGES>
__device__ __forceinline__ void kv4_many_block(const Kv4View& c, const Kv4Rows& b, const Kv4Attn& a, Kv4ManyLds<HD>& lds, int h, int turn, int seq) {
    uint8_t (&kbuf)[2][128 * HD] = lds.k;
    uint8_t (&vbuf)[2][128 * HD] = lds.v;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    const Kv4Seq s = kv4_seq_of(b, c, seq);
    const int rows = s.n < b.max_rows ? s.n : b.max_rows, cols = rows * a.group;
    if (s.state == 1 || cols <= KV4_FEW_COLUMNS) return;
    // the last tiles see most: they start first
    constexpr int COLS = 64 * NC;
    const int block = (cols + COLS - 1) / COLS - 1 - turn;
    if (block < 0) return;
    const int c0 = (block * 4 + w) * (16 * NC), c1 = cols < c0 + 16 * NC ? cols : c0 + 16 * NC;
    if (s.state == 2) {
        if (c0 < cols) kv4_fill_columns<HD>(a, s, h, c0, c1, lane, 64);
        return;
    }
    Kv4Query<HD, F16> q[NC];
    int sees[NC], seen[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int col = c0 + 16 * n + (lane & 15), j = a.row(col);
        q[n].load(col < c1 ? a.q_at(s.start + j, (h * a.group + col - j * a.group) * HD) : nullptr, lane,
                  a.frags && c0 + 16 * n < c1 ? a.frags + (kv4_column(a, h, seq, s) + c0 + 16 * n) * (2 * HD) : nullptr);
        sees[n] = col < c1 ? s.ctx - s.n + j + 1 : 0;
    }
    // what the wave's first and last row see; a wave without columns sees nothing and only converts
    const int base = s.ctx - s.n + 1, least = base + a.row(c0), most = c0 < cols ? base + a.row(c1 - 1) : 0;
    const int end = block * COLS + COLS, all = base + a.row((cols < end ? cols : end) - 1);      // the workgroup's last row
    Kv4State<HD, NC> st;
    st.clear();
    const int32_t* bt = c.table + (int64_t)s.stream * c.max_pages;
    const int pages = all > 0 ? (all + KV4_PAGE - 1) / KV4_PAGE : 0;
    const int mine = most > 0 ? (most + KV4_PAGE - 1) / KV4_PAGE : 0;        // pages that the wave looks at
    const auto page_id = [&](int p) { return __builtin_amdgcn_readfirstlane(bt[p < pages ? p : pages - 1]); };
    // a page on its way to its half of the buffer: load() sets out, store() is done when it has arrived
    Kv4Stage<HD> stage;
    int id = pages > 0 && !IMAGES ? page_id(0) : 0;
    const auto load = [&](int p) {
        if constexpr (IMAGES) {
            if (p < pages) kv4_image_to_lds<HD>(kv4_image<HD>(a, c.Hkv, seq, h, p), kbuf[p & 1], vbuf[p & 1], w, lane);
        } else {
            stage.load_k(c, id, h, w, lane);
            stage.load_v(c, id, h, w, lane);
            id = page_id(p + 1);
        }
    };
    const auto store = [&](int p) {
        if constexpr (IMAGES) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        } else {
            stage.store_k(kbuf[p & 1], w, lane);
            stage.store_v(vbuf[p & 1], s.ctx - p * KV4_PAGE, w, lane);
        }
    };
    if (pages > 0) { load(0); store(0); }
    __syncthreads();
    int p = 0;
    for (; p < mine; ++p) {
        const int first = p * KV4_PAGE;
        load(p + 1);
        f32x4 sc[NC][4];
        bf16x8 ph[NC][2], pl[NC][2];
        kv4_lds_scores<HD, F16, NC>(kbuf[p & 1], q, sc, lane);
        kv4_interleave<HD / 8, NC * (F16 ? 2 : 1)>();
        if (least < first + KV4_PAGE) {
#pragma unroll
            for (int n = 0; n < NC; ++n) seen[n] = sees[n] - first;
            kv4_hide_scores<NC>(sc, seen, lane);
        }
        kv4_reference<HD, NC>(sc, st, a.c);
        kv4_probabilities<HD, NC, F16>(sc, st, a.c, ph, pl);
        __builtin_amdgcn_sched_barrier(0);
        kv4_lds_values<HD, F16, NC>(vbuf[p & 1], ph, pl, st, lane);
        kv4_interleave<HD / 8, NC * (F16 ? 2 : 1)>();
        __builtin_amdgcn_sched_barrier(0);
        store(p + 1);
        __syncthreads();
    }
    // pages that only later waves of the workgroup see
    for (; p < pages; ++p) {
        load(p + 1);
        store(p + 1);
        __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int col = c0 + 16 * n + (lane & 15), j = a.row(col), head = h * a.group + col - j * a.group;
        const float l = kv4_group_sum(st.l[n]);
        if (col >= c1) continue;
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        uint16_t* op = a.out_at(s.start + j, head * HD + 16 * g);
#pragma unroll
        for (int x = 0; x < HD / 64; ++x)
#pragma unroll
            for (int jj = 0; jj < 4; jj += 2) {
                const f32x4 (&o)[4] = st.o[n][x];
                const u32x4 r = {kv4_pack2<F16>(o[0][jj] * inv, o[1][jj] * inv), kv4_pack2<F16>(o[2][jj] * inv, o[3][jj] * inv),
                                 kv4_pack2<F16>(o[0][jj + 1] * inv, o[1][jj + 1] * inv), kv4_pack2<F16>(o[2][jj + 1] * inv, o[3][jj + 1] * inv)};
                *reinterpret_cast<u32x4*>(op + 64 * x + 4 * jj) = r;
            }
        if (a.norm && g == 0) a.norm[kv4_column(a, h, seq, s) + col] = f32x2{st.m[n], inv};
    }
}

// Both in one launch, for a batch that may hold sequences of either kind: the long blocks start first.
template <int HD, bool F16, int NC, bool IMAGES>
__global__ __launch_bounds__(256, HD == 64 ? 4 : 2) void kv4_attn_mixed_kernel(Kv4View c, Kv4Rows b, Kv4Attn a, int turns, unsigned first) {
    __shared__ union { Kv4ManyLds<HD> many; Kv4FewLds<HD> few; } lds;
    const unsigned many = (unsigned)c.Hkv * turns * b.n_seqs;
    unsigned x = first + blockIdx.x;
    if (x < many) {
        const int h = x % c.Hkv;
        x /= c.Hkv;
        kv4_many_block<HD, F16, NC, IMAGES>(c, b, a, lds.many, h, x % turns, x / turns);
    } else {
        x -= many;
        const int h = x % c.Hkv;
        x /= c.Hkv;
        const int tile = x % a.tiles;
        x /= a.tiles;
        kv4_few_block<HD, F16, false>(c, b, a, lds.few, h, tile, x % b.n_seqs, x / b.n_seqs);
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Weights: W[stream][key head][t] += sum over the sequence's columns of exp2((s - m) c) / l.  A workgroup owns its entries and walks the
// columns in a fixed order, so there are no atomics.  Scores of sequences of few columns were kept by the pass above (64 decode rows x
// 16 heads of 64 over up to 2000 entries 55 us -> 37, 32 x 64 heads on 8 of 128 over up to 8000 122 -> 74; 40 columns 37 -> 28); the
// others are formed again from K, from queries that the pass above leaves in operand order (2 x 4095 rows x 32 heads of 128: 312 us
// beside the pass's 351; from the rows as given 100 us more, by one wave a page 890).
// A stream that occurs in several sequences of the call is done, in their order, by the waves of the first of them.
// ------------------------------------------------------------------------------------------------------------------
// Walks the sequences of the stream of sequence `seq` if that is the first of them, 64 looked at at a time: fn(their numbers).
// False if an earlier one is, or if there is no such stream.
template <typename Fn> __device__ __forceinline__ bool kv4_of_stream(const Kv4Rows& b, const Kv4View& c, int seq, int lane, Fn fn) {
    const Kv4Seq own = kv4_seq_of(b, c, seq);
    if (own.stream < 0 || own.stream >= c.n_streams) return false;
    for (int i0 = 0; i0 < b.n_seqs; i0 += 64) {
        uint64_t todo = __ballot(i0 + lane < b.n_seqs && b.stream[i0 + lane < b.n_seqs ? i0 + lane : seq] == own.stream);
        for (; todo; todo &= todo - 1) {
            const int i = i0 + __builtin_ctzll(todo);
            if (i < seq) return false;
            Kv4Seq s = own;
            if (i != seq) s = kv4_seq_of(b, c, i);
            fn(i, s);
        }
    }
    return true;
}

// Every sequence of the call has its scores kept.  A thread has four entries; with GROUPS = 4 the workgroup's waves take every
// fourth column each of the same entries and are added in order (the order of the single one while there are at most 4 columns).
// The columns' m and l are joined here from their chunks', so that this runs beside the join of the outputs, in one launch: 9 to 10 us
// at 64 x 16 heads x 300..2000 entries, latency (a chain of six loads and barriers at 32 waves a CU).
template <int GROUPS> struct Kv4KeptLds {
    f32x2 part[256], norm[KV4_FEW_COLUMNS];
    f32x4 sum[GROUPS][64];
};
template <int GROUPS>
__device__ __forceinline__ void kv4_kept_block(const Kv4View& c, const Kv4Rows& b, const Kv4Attn& a, Kv4KeptLds<GROUPS>& lds, float* weights,
                                               int64_t weights_stride, int h, int piece, int seq) {
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int from = piece * (GROUPS == 1 ? 1024 : 256), first = from + (GROUPS == 1 ? tid : lane) * 4;
    f32x4 mine = {0.f, 0.f, 0.f, 0.f};
    const bool own = kv4_of_stream(b, c, seq, lane, [&](int i, const Kv4Seq& s) {
        if (s.state || from >= s.ctx) return;                     // (for all threads)
        const int rows = s.n < b.max_rows ? s.n : b.max_rows, cols = rows * a.group, chunks = kv4_chunks(s.ctx);
        // m and 1 / l: 16, 8 or 4 threads a column, every so many chunks each
        const int log = cols <= 16 ? 4 : cols <= 32 ? 3 : 2, each = tid >> log;
        float M = KV4_NONE, L = 0.f;
        if (each < cols) {
            const f32x2* ml = a.ml + kv4_states_at(a, h, i, s, each);
            for (int x = tid & ((1 << log) - 1); x < chunks; x += 1 << log) {
                const f32x2 part = ml[x];
                const float top = fmaxf(M, part[0]);
                L = fmaf(L, kv4_exp(M, top, a.c), part[1] * kv4_exp(part[0], top, a.c));
                M = top;
            }
        }
        lds.part[tid] = f32x2{M, L};
        __syncthreads();
        if (tid < cols) {
            M = KV4_NONE;
            L = 0.f;
            for (int x = tid << log; x < (tid + 1) << log; ++x) M = fmaxf(M, lds.part[x][0]);
            for (int x = tid << log; x < (tid + 1) << log; ++x) L = fmaf(lds.part[x][1], kv4_exp(lds.part[x][0], M, a.c), L);
            lds.norm[tid] = f32x2{M, L == 0.f ? 0.f : 1.0f / L};
        }
        __syncthreads();
        if (first >= s.ctx) return;
        const int64_t width = kv4_kept_width(s.ctx);
        const float* sp = kv4_scores_at(a, h, i, s) + first;
#pragma unroll 4
        for (int col = GROUPS == 1 ? 0 : w; col < cols; col += GROUPS) {
            const int seen = s.ctx - s.n + a.row(col) + 1 - first;
            const f32x2 norm = lds.norm[col];
            const f32x4 x = *reinterpret_cast<const f32x4*>(sp + col * width);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v = kv4_exp(x[e], norm[0], a.c);
                mine[e] += e < seen ? v * norm[1] : 0.f;
            }
        }
    });
    if (!own) return;                                             // the same in all waves
    if constexpr (GROUPS > 1) {
        lds.sum[w][lane] = mine;
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int x = 1; x < GROUPS; ++x) mine += lds.sum[x][lane];
    }
    float* wp = weights + ((int64_t)b.stream[seq] * c.Hkv + h) * weights_stride + first;
    const bool any = mine[0] != 0.f || mine[1] != 0.f || mine[2] != 0.f || mine[3] != 0.f;   // else nothing is touched
    if (weights_stride % 4 == 0 && reinterpret_cast<uintptr_t>(weights) % 16 == 0) {
        if (any && first < weights_stride) {
            f32x4 v = *reinterpret_cast<const f32x4*>(wp);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = mine[e] != 0.f ? v[e] + mine[e] : v[e];
            *reinterpret_cast<f32x4*>(wp) = v;
        }
    } else if (any) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (mine[e] != 0.f && first + e < weights_stride) wp[e] += mine[e];
    }
}
// blocks of a sequence: `joins` columns x key heads of the outputs' join, then its pieces of entries x key heads
template <int HD, bool F16, int GROUPS>
__global__ __launch_bounds__(256, 8) void kv4_finish_kernel(Kv4View c, Kv4Rows b, Kv4Attn a, float* weights, int64_t weights_stride, int joins) {
    __shared__ __attribute__((aligned(16))) union { Kv4JoinLds<HD> join; Kv4KeptLds<GROUPS> kept; } lds;
    const bool join = (int)blockIdx.x < joins;
    const int x = join ? blockIdx.x : blockIdx.x - joins, y = x / c.Hkv, h = x - y * c.Hkv;
    if (join) kv4_join_block<HD, F16>(c, b, a, lds.join, h, y, blockIdx.y);
    else kv4_kept_block<GROUPS>(c, b, a, lds.kept, weights, weights_stride, h, y, blockIdx.y);
}

// Some have not: a workgroup per (page, key head, stream).  A wave keeps the page's keys as operands, takes every fourth column tile
// (the next one's queries are under way meanwhile) and sums over its tiles and their columns; the waves are added in order.  At hd 128 two
// workgroups a CU share its L1 better than the three that the registers leave room for: 2 x 4095 rows x 32 heads with weights 663 us
// and 713; at hd 64 four are better than two, 4 x 2000 rows x 16 heads 111 and 118.
template <int HD, bool F16>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, HD == 64 ? 4 : 2))) void kv4_weights_kernel(Kv4View c, Kv4Rows b, Kv4Attn a, float* weights, int64_t weights_stride) {
    __shared__ float part[4][KV4_PAGE];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
    const int h = blockIdx.y, seq = blockIdx.z, p = blockIdx.x, first = p * KV4_PAGE;
    bf16x8 kf[4][HD / 32];
    bool have = false;
    float mine = 0.f;                                             // of token first + lane
    const bool own = kv4_of_stream(b, c, seq, lane, [&](int i, const Kv4Seq& s) {
        if (s.state || first >= s.ctx) return;
        const int rows = s.n < b.max_rows ? s.n : b.max_rows, cols = rows * a.group;
        if (kv4_kept(cols, s.ctx, a.room)) {
            const int64_t width = kv4_kept_width(s.ctx);
            const float* sp = kv4_scores_at(a, h, i, s) + first + lane;
            for (int col = w; col < cols; col += 4) {
                const int j = a.row(col);
                const f32x2 norm = a.norm[kv4_column(a, h, i, s) + col];
                const float v = kv4_exp(sp[col * width], norm[0], a.c);
                mine += first + lane < s.ctx - s.n + j + 1 ? v * norm[1] : 0.f;
            }
            return;
        }
        if (!have) {
            Kv4Page<HD> pg;
            kv4_fetch_k<HD, false>(pg, c, __builtin_amdgcn_readfirstlane(c.table[(int64_t)s.stream * c.max_pages + p]), h, lane);
            kv4_operands<HD>(pg, kf);
            have = true;
        }
        float sum[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) sum[e] = 0.f;
        // rows before the first that sees this page add nothing
        const int base = s.ctx - s.n + 1, j0 = first + 1 - base;
        const int t0 = j0 > 0 ? j0 * a.group / 16 : 0, tiles = (cols + 15) / 16;
        // the tiles' queries as the pass above left them (54 cache lines' lookups a load become 16) and their columns' norms
        const int64_t column = kv4_column(a, h, i, s);
        const uint8_t* qp = a.frags + column * (2 * HD) + lane * 16;
        const f32x2* np = a.norm + column + (lane & 15);
        struct Tile { u32x4 q[HD / 32]; f32x2 norm; int col; } even, odd;
        const auto fetch = [&](Tile& t, int tile) {
#pragma unroll
            for (int x = 0; x < HD / 32; ++x) t.q[x] = *reinterpret_cast<const u32x4*>(qp + (int64_t)tile * (32 * HD) + x * 1024);
            t.norm = np[tile * 16];
            t.col = tile * 16 + (lane & 15);
        };
        const auto add = [&](const Tile& t) {
            Kv4Query<HD, F16> q;
#pragma unroll
            for (int x = 0; x < HD / 32; ++x) q.set(x, t.q[x]);
            const int seen = t.col < cols ? base + a.row(t.col) - first - 16 * g : 0;      // of the lane's 16 tokens
            f32x4 sc[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < HD / 32; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i][x], q.q[x], sc[i], 0, 0, 0);
                    if constexpr (F16) sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[i][x], q.q[HD / 32 + x], sc[i], 0, 0, 0);
                }
            if (__all(seen >= 16)) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    sum[e] = fmaf(kv4_exp(sc[e & 3][e >> 2], t.norm[0], a.c), t.norm[1], sum[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float v = kv4_exp(sc[e & 3][e >> 2], t.norm[0], a.c);
                    sum[e] = e < seen ? fmaf(v, t.norm[1], sum[e]) : sum[e];
                }
            }
        };
        int tile = t0 + w;
        if (tile < tiles) fetch(even, tile);
        for (; tile < tiles; tile += 8) {
            fetch(odd, tile + 4 < tiles ? tile + 4 : tile);
            add(even);
            fetch(even, tile + 8 < tiles ? tile + 8 : tile);
            if (tile + 4 < tiles) add(odd);
        }
        // over the 16 columns; lane r of a group takes token 16 g + r
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float all = kv4_row_sum(sum[e]);
            mine += (lane & 15) == e ? all : 0.f;
        }
    });
    if (!own) return;                                             // the same in all waves
    part[w][lane] = mine;
    __syncthreads();
    const int64_t t = first + lane;
    if (w == 0 && t < weights_stride) {
        const float all = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
        float* wp = weights + ((int64_t)b.stream[seq] * c.Hkv + h) * weights_stride + t;
        if (all != 0.f) *wp += all;
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Entry points
// ------------------------------------------------------------------------------------------------------------------
// the work buffer: chunks' O | their m and l | kept scores | m and 1 / l | queries | converted pages
struct Kv4Work {
    int64_t states, ml, scores, norm, frags, images, room, kept_unit;
    Kv4Place few, kept;
    int tiles, chunks, slots, pages;
    int64_t bytes() const { return states + ml + scores + norm + frags + images; }
};
// Pages are converted by a launch of their own from this many columns on (6 x 513 rows x 16 heads of 64 18.0 us, so 18.4; 4 x 1000 34.3 and
// 28.9; 64 x 100 41 and 60), unless they need more than this many bytes
#define KV4_IMAGE_COLUMNS 768
#define KV4_IMAGE_BYTES (1ll << 29)
static Kv4Work plan_work(const t3_kv4_cache* c, const t3_kv4_batch* b, int H, bool weights) {
    Kv4Work w{};
    const int64_t group = H / c->Hkv, cols = b->max_rows * group, few = cols < KV4_FEW_COLUMNS ? cols : KV4_FEW_COLUMNS;
    const int64_t cap = (int64_t)c->max_pages * KV4_PAGE, most = b->max_ctx < cap ? b->max_ctx : cap, pairs = (int64_t)b->n_seqs * c->Hkv;
    const auto whole = [](int64_t bytes) { return (bytes + 255) / 256 * 256; };
    w.tiles = (int)((few + 15) / 16);
    w.chunks = kv4_chunks((int)most);
    // columns of sequences of few: not more than the rows have, nor than `few` a sequence
    const int64_t by_row = b->rows * group, by_seq = b->n_seqs * few, columns = by_row < by_seq ? by_row : by_seq;
    const auto by_rows = [&] { return Kv4Place{0, 0, (unsigned)(c->Hkv * group), (unsigned)group}; };
    w.few = by_row < by_seq ? by_rows() : Kv4Place{(unsigned)(c->Hkv * few), (unsigned)few, 0, 0};
    const int64_t parts = c->Hkv * columns * w.chunks;
    w.states = w.chunks > 1 ? whole(parts * c->hd * 4) : 0;
    w.ml = w.chunks > 1 ? whole(parts * 8) : 0;
    if (weights) {
        const int64_t width = kv4_kept_width(most), every = few * width;
        w.room = every < KV4_KEEP ? every : KV4_KEEP;
        // by rows; by sequences; by sequences with less room for each, so that fewer have their scores kept
        if (by_row * width < b->n_seqs * w.room && c->Hkv * by_row * width * 4 <= KV4_KEEP_BYTES) {
            w.kept = by_rows();
            w.kept_unit = width;
            w.scores = c->Hkv * by_row * width * 4;
        } else {
            if (pairs * w.room * 4 > KV4_KEEP_BYTES) w.room = KV4_KEEP_BYTES / 4 / pairs / KV4_PAGE * KV4_PAGE;
            w.kept = Kv4Place{(unsigned)c->Hkv, 1, 0, 0};
            w.kept_unit = w.room;
            w.scores = pairs * w.room * 4;
        }
        w.slots = (int)(by_row / 16) + b->n_seqs + 1;
        if (cols > few || every > w.room) {                       // some scores are formed again
            w.norm = (int64_t)c->Hkv * w.slots * 16 * 8;
            w.frags = (int64_t)c->Hkv * w.slots * 16 * c->hd * 2;
        } else {
            w.ml = whole(parts * 8);
        }
    }
    w.pages = (int)((most + KV4_PAGE - 1) / KV4_PAGE);
    w.images = pairs * w.pages * 256 * c->hd;
    if (cols < KV4_IMAGE_COLUMNS || cols <= few || w.images > KV4_IMAGE_BYTES) w.images = 0;
    return w;
}
static int check_sizes(const t3_kv4_cache* c, const t3_kv4_batch* b, int H) {
    T3_REQUIRE(b->max_ctx <= (1 << 26) || c->max_pages <= (1 << 26) / KV4_PAGE, "attn_kv4: more than 2^26 entries in a stream");
    T3_REQUIRE(H >= c->Hkv && H % c->Hkv == 0 && H / c->Hkv <= 64, "attn_kv4: query heads must be 1..64 times the key heads");
    T3_REQUIRE((int64_t)b->max_rows * (H / c->Hkv) <= (1 << 22), "attn_kv4: more than 2^22 rows x query heads of a key head");
    T3_REQUIRE((int64_t)b->rows * (H / c->Hkv) <= (1 << 30), "attn_kv4: more than 2^30 rows x query heads of a key head in one call");
    return 0;
}

extern "C" int64_t t3_op_attn_kv4_work_bytes(const t3_kv4_cache* cache, const t3_kv4_batch* batch, int32_t H, int32_t with_weights) {
    if (kv4_check_cache(cache, 0, 1, nullptr) || kv4_check_batch(batch) || check_sizes(cache, batch, H)) return -1;
    const Kv4Work w = plan_work(cache, batch, H, with_weights != 0);
    return w.bytes();
}

// The launch for few columns has its chunks along the grid's third axis, which ends at 65535; one for both kinds, and none of the other,
// takes more.  That has at most KV4_LAUNCH_BLOCKS workgroups (a grid's threads end at 2^32); what is more goes into further ones.
#define KV4_LAUNCH_CHUNKS 65535
#define KV4_LAUNCH_BLOCKS (1ll << 23)
template <int HD, bool F16>
static int launch_attn(const Kv4View& c, const Kv4Rows& b, const Kv4Attn& a, float* weights, int64_t weights_stride, hipStream_t st) {
    // column tiles of a wave: at hd 128 two share each fragment's way through LDS (372 us; one, with eight waves a workgroup, 395); at
    // hd 64 one leaves room for four waves a SIMD instead of two (4 x 2000 rows 70.6 us; two 78, four 98)
    constexpr int NC = HD == 64 ? 1 : 2;
    const int64_t cols = (int64_t)b.max_rows * a.group;
    if (cols <= KV4_FEW_COLUMNS && a.chunks <= KV4_LAUNCH_CHUNKS) {
        const dim3 grid(a.tiles * c.Hkv, b.n_seqs, a.chunks);
        if (a.tiles == 1) T3_LAUNCH((kv4_attn_few_kernel<HD, F16, true>), grid, dim3(64 * KV4_FEW_WAVES), 0, st, c, b, a);
        else T3_LAUNCH((kv4_attn_few_kernel<HD, F16, false>), grid, dim3(64 * KV4_FEW_WAVES), 0, st, c, b, a);
    } else {
        const int64_t turns = cols > KV4_FEW_COLUMNS ? (cols + 64 * NC - 1) / (64 * NC) : 0, blocks = c.Hkv * (int64_t)b.n_seqs * (turns + (int64_t)a.tiles * a.chunks);
        T3_REQUIRE(blocks <= INT32_MAX, "attn_kv4: too many sequences of that many rows in one call");
        if (a.images) T3_LAUNCH(kv4_image_kernel<HD>, dim3(a.pages * c.Hkv, b.n_seqs), dim3(256), 0, st, c, b, a);
        for (int64_t first = 0; first < blocks; first += KV4_LAUNCH_BLOCKS) {
            const dim3 grid((unsigned)(blocks - first < KV4_LAUNCH_BLOCKS ? blocks - first : KV4_LAUNCH_BLOCKS));
            if (a.images) T3_LAUNCH((kv4_attn_mixed_kernel<HD, F16, NC, true>), grid, dim3(256), 0, st, c, b, a, (int)turns, (unsigned)first);
            else T3_LAUNCH((kv4_attn_mixed_kernel<HD, F16, NC, false>), grid, dim3(256), 0, st, c, b, a, (int)turns, (unsigned)first);
        }
    }
    const int joins = a.chunks > 1 ? (cols < KV4_FEW_COLUMNS ? (int)cols : KV4_FEW_COLUMNS) * c.Hkv : 0;
    const int64_t cap = (int64_t)c.max_pages * KV4_PAGE, most = b.max_ctx < cap ? b.max_ctx : cap;
    if (weights && !a.frags) {
        if (cols <= 4)
            T3_LAUNCH((kv4_finish_kernel<HD, F16, 1>), dim3((unsigned)(joins + (most + 1023) / 1024 * c.Hkv), b.n_seqs), dim3(256), 0, st,
                      c, b, a, weights, weights_stride, joins);
        else
            T3_LAUNCH((kv4_finish_kernel<HD, F16, 4>), dim3((unsigned)(joins + (most + 255) / 256 * c.Hkv), b.n_seqs), dim3(256), 0, st,
                      c, b, a, weights, weights_stride, joins);
    } else {
        if (joins) T3_LAUNCH((kv4_attn_join_kernel<HD, F16>), dim3(joins, b.n_seqs), dim3(256), 0, st, c, b, a);
        if (weights)
            T3_LAUNCH((kv4_weights_kernel<HD, F16>), dim3((unsigned)((most + KV4_PAGE - 1) / KV4_PAGE), c.Hkv, b.n_seqs), dim3(256), 0, st,
                      c, b, a, weights, weights_stride);
    }
    T3_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int t3_op_attn_kv4(const t3_kv4_cache* cache, const t3_kv4_batch* batch, const void* q_dev, int64_t q_stride,
                              void* out_dev, int64_t out_stride, int32_t H, int32_t dtype, float scale, float* weights_dev,
                              int64_t weights_stride, void* work_dev, int64_t work_bytes, int32_t layer, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (kv4_check_cache(cache, layer, 1, st) || kv4_check_batch(batch) || check_sizes(cache, batch, H)) return 1;
    T3_REQUIRE(q_dev && out_dev, "attn_kv4: null argument");
    T3_REQUIRE(dtype == 0 || dtype == 1, "attn_kv4: dtype must be 0 (bf16) or 1 (fp16)");
    T3_REQUIRE(scale > 0.f && scale < 1e8f, "attn_kv4: scale must be positive");
    const int64_t width = (int64_t)H * cache->hd;
    T3_REQUIRE(q_stride >= width && out_stride >= width && q_stride % 8 == 0 && out_stride % 8 == 0 &&
               reinterpret_cast<uintptr_t>(q_dev) % 16 == 0 && reinterpret_cast<uintptr_t>(out_dev) % 16 == 0,
               "attn_kv4: rows must be 16-byte aligned and must not overlap");
    T3_REQUIRE(q_stride <= INT32_MAX && out_stride <= INT32_MAX, "attn_kv4: row stride of more than 2^31 elements");
    T3_REQUIRE(!weights_dev || weights_stride >= batch->max_ctx, "attn_kv4: weights_stride must be at least max_ctx");
    const int64_t needed = t3_op_attn_kv4_work_bytes(cache, batch, H, weights_dev != nullptr);
    T3_REQUIRE(needed == 0 || (work_dev && work_bytes >= needed && reinterpret_cast<uintptr_t>(work_dev) % 16 == 0),
               "attn_kv4: the work buffer is too small or not 16-byte aligned");
    Kv4Attn a{};
    a.q = static_cast<const uint16_t*>(q_dev); a.q_stride = (unsigned)q_stride;
    a.out = static_cast<uint16_t*>(out_dev); a.out_stride = (unsigned)out_stride;
    a.group = H / cache->Hkv;
    a.inv = a.group == 1 ? 0u : (unsigned)(((1ull << 32) + a.group - 1) / a.group);
    a.c = scale * 1.44269504088896340736f;
    const Kv4Work w = plan_work(cache, batch, H, weights_dev != nullptr);
    uint8_t* work = static_cast<uint8_t*>(work_dev);
    a.tiles = w.tiles; a.chunks = w.chunks; a.room = w.room; a.few = w.few; a.kept = w.kept; a.kept_unit = w.kept_unit;
    a.states = reinterpret_cast<float*>(work);
    work += w.states;
    a.ml = w.ml ? reinterpret_cast<f32x2*>(work) : nullptr;
    work += w.ml;
    a.scores = w.scores ? reinterpret_cast<float*>(work) : nullptr;
    work += w.scores;
    a.norm = w.norm ? reinterpret_cast<f32x2*>(work) : nullptr;
    a.frags = w.frags ? work + w.norm : nullptr;
    work += w.norm + w.frags;
    a.images = w.images ? work : nullptr;
    a.pages = w.pages;
    a.slots = w.slots;
    const Kv4View c = kv4_view(cache, layer);
    const Kv4Rows b = kv4_rows(batch);
    if (cache->hd == 64) return dtype ? launch_attn<64, true>(c, b, a, weights_dev, weights_stride, st) : launch_attn<64, false>(c, b, a, weights_dev, weights_stride, st);
    return dtype ? launch_attn<128, true>(c, b, a, weights_dev, weights_stride, st) : launch_attn<128, false>(c, b, a, weights_dev, weights_stride, st);
}
