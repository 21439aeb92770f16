// Attention over the 4-bit KV cache (byte order: kv4_layout.h).
//
// A column is a (row, query head) pair; the group = H / Hkv query heads of a key head and the rows of a sequence share its keys,
// so column c of a sequence and key head is row c / group, head c % group, and 16 columns make one tile of
//   S^T[token][column] = K Q^T        K codes -> bf16 in registers (exact), Q held in registers for the whole pass
//   O^T[dim][column]   = V^T P^T      P as bf16 hi + lo parts, so the probabilities keep 16 significant bits
// on v_mfma_f32_16x16x32_bf16, a page of 64 tokens at a time.  A lane ends the first product with 16 consecutive tokens of one
// column, which is what the second takes from it: no exchange but the maximum over the four lane groups.
// fp16 queries enter as bf16 hi + lo (exact to 2^-16 of the value, fp16 has 11 bits), so one set of products serves both types.
//
//   p = exp2(s c - m),  c = scale log2(e),  m the running maximum of s c as rounded, l the running sum:  one pass, fp32.
// Keeping m as the rounded product makes the factors between pages and chunks, exp2(m - m'), consistent at any size of s.
//
// Sequences of at most KV4_FEW_COLUMNS columns (decode steps, drafted tokens) are cut into chunks of their cache, a workgroup of
// four waves each; a second launch joins the chunks in order.  The chunk length follows from the sequence's own length, so a
// row's bits do not depend on the batch.  Longer ones (prompts) run whole: a wave keeps four column tiles and walks the cache.
#include "kv4_common.h"

#define KV4_FEW_COLUMNS 64        // rows x group up to which a sequence is cut along its cache
#define KV4_NONE -1e30f           // running maximum before the first visible token

// pages of a chunk
KV4_FN int kv4_chunk_pages(int ctx) { return ctx > 8192 ? 16 : 8; }
KV4_FN int kv4_chunks(int ctx) { const int p = (ctx + KV4_PAGE - 1) / KV4_PAGE, n = kv4_chunk_pages(ctx); return (p + n - 1) / n; }
KV4_FN int kv4_max_chunks(int max_ctx) {                 // over all lengths up to max_ctx
    const int a = kv4_chunks(max_ctx < 8192 ? max_ctx : 8192), b = kv4_chunks(max_ctx);
    return a > b ? a : b;
}

struct Kv4Attn {
    const uint16_t* q; int64_t q_stride;
    uint16_t* out; int64_t out_stride;
    int group, tiles, chunks;     // query heads per key head; column tiles and chunks the state buffer holds per (sequence, key head)
    float c;                      // scale * log2(e)
    float* states;                // [sequence][key head][tile][chunk] x kv4_state_floats
    f32x2* norm;                  // [rows][H]: m and 1 / l of each column, or null
};
// state of (chunk, tile): m[16], l[16], O[16][hd]
template <int HD> __device__ __forceinline__ int64_t kv4_state_at(const Kv4Attn& a, int Hkv, int seq, int h, int tile, int chunk) {
    return ((((int64_t)seq * Hkv + h) * a.tiles + tile) * a.chunks + chunk) * (16 * (HD + 2));
}

template <int HD> struct Kv4Page {
    u32x4 k[HD / 32], v[HD / 32], vs[HD / 64];
    unsigned ks;
    __device__ __forceinline__ void load(const uint8_t* slab, int lane) {
        const int g = lane >> 4, r = lane & 15;
#pragma unroll
        for (int x = 0; x < HD / 32; ++x) k[x] = *reinterpret_cast<const u32x4*>(slab + x * 1024 + lane * 16);
        ks = *reinterpret_cast<const unsigned*>(slab + 64 * HD + g * (HD / 4) / KV4_BLOCK * KV4_PAGE + 4 * r);
#pragma unroll
        for (int x = 0; x < HD / 32; ++x) v[x] = *reinterpret_cast<const u32x4*>(slab + 32 * HD + x * 1024 + lane * 16);
#pragma unroll
        for (int x = 0; x < HD / 64; ++x) vs[x] = *reinterpret_cast<const u32x4*>(slab + 66 * HD + (2 * x + (r >> 3)) * KV4_PAGE + 16 * g);
    }
};
__device__ __forceinline__ unsigned kv4_byte(unsigned w, int i) { return w >> (8 * i) & 255u; }

// Q of one column tile: step x of the product takes dims g hd/4 + 8 x .. + 7 of lane group g
template <int HD, bool F16> struct Kv4Query {
    bf16x8 q[(F16 ? 2 : 1) * HD / 32];
    __device__ __forceinline__ void load(const uint16_t* row, int lane) {          // null: a column that is none
        const int g = lane >> 4;
#pragma unroll
        for (int x = 0; x < HD / 32; ++x) {
            u32x4 w = {0u, 0u, 0u, 0u};
            if (row) w = *reinterpret_cast<const u32x4*>(row + g * (HD / 4) + 8 * x);
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
    }
};

// S^T of a page for NC column tiles: s[n][i][j] = token 16 g + 4 j + i, column lane & 15
template <int HD, bool F16, int NC>
__device__ __forceinline__ void kv4_scores(const Kv4Page<HD>& pg, const Kv4Query<HD, F16> (&q)[NC], f32x4 (&s)[NC][4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float sc = kv4_scale(kv4_byte(pg.ks, i));
#pragma unroll
        for (int n = 0; n < NC; ++n) s[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < HD / 32; ++x) {
            const unsigned w = HD == 64 ? pg.k[i / 2][i % 2 * 2 + x] : pg.k[HD == 64 ? 0 : i][x];
            const u32x4 a = {kv4_pair<0>(w, sc), kv4_pair<1>(w, sc), kv4_pair<2>(w, sc), kv4_pair<3>(w, sc)};
            const bf16x8 af = __builtin_bit_cast(bf16x8, a);
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                s[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, q[n].q[x], s[n][i], 0, 0, 0);
                if constexpr (F16) s[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af, q[n].q[HD / 32 + x], s[n][i], 0, 0, 0);
            }
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

// One page.  seen[n]: tokens of this page that column tile n's column sees (>= 64: all); tail: tokens of the page that exist.
template <int HD, bool F16, int NC, bool MASK>
__device__ __forceinline__ void kv4_page_step(const Kv4Page<HD>& pg, const Kv4Query<HD, F16> (&q)[NC], Kv4State<HD, NC>& st,
                                              const int (&seen)[NC], int tail, float c, int lane) {
    const int g = lane >> 4;
    f32x4 s[NC][4];
    kv4_scores<HD, F16, NC>(pg, q, s);
    bf16x8 ph[NC][2], pl[NC][2];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        if constexpr (MASK) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[n][i][j] = 16 * g + 4 * j + i < seen[n] ? s[n][i][j] : -INFINITY;
        }
        float top = s[n][0][0];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) top = fmaxf(top, s[n][i][j]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float m = fmaxf(st.m[n], top * c), alpha = __builtin_amdgcn_exp2f(st.m[n] - m);
        st.m[n] = m;
        float sum = 0.f;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < 8; ++y) {
                const int e = 8 * x + y;                          // token 16 g + e
                const float p = __builtin_amdgcn_exp2f(fmaf(s[n][e & 3][e >> 2], c, -m));
                sum += p;
                const __bf16 hi = (__bf16)p;
                ph[n][x][y] = hi;
                pl[n][x][y] = (__bf16)(p - (float)hi);
            }
        st.l[n] = fmaf(st.l[n], alpha, sum);
#pragma unroll
        for (int h = 0; h < HD / 64; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) st.o[n][h][e] *= alpha;
    }
#pragma unroll
    for (int h = 0; h < HD / 64; ++h)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            u32x4 a[4];                                           // tile e: 8 tokens of dim 64 h + 4 r + e
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const unsigned codes = pg.v[2 * h + x][w];
                const int t = 8 * x + 2 * w;                      // tokens 16 g + t, + t + 1
                unsigned b0 = kv4_byte(pg.vs[h][t / 4], t % 4), b1 = kv4_byte(pg.vs[h][t / 4], t % 4 + 1);
                if constexpr (MASK) {                             // what lies behind the last entry may be anything: 0 * finite
                    b0 = 16 * g + t < tail ? b0 : 0u;
                    b1 = 16 * g + t + 1 < tail ? b1 : 0u;
                }
                const float s0 = kv4_scale(b0), s1 = kv4_scale(b1);
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

template <bool F16> __device__ __forceinline__ unsigned kv4_pack2(float lo, float hi) {
    if constexpr (F16) {
        const f16x2 p = {(_Float16)lo, (_Float16)hi};
        return __builtin_bit_cast(unsigned, p);
    } else {
        return pack_bf2(lo, hi);
    }
}
// A page of a stream.  An id outside the pool is not followed: the page then holds NaN keys, and values that a row which does not
// see it can multiply by zero.
template <int HD> __device__ __forceinline__ void kv4_fetch(Kv4Page<HD>& pg, const Kv4View& c, const int32_t* bt, int p, int h, int lane) {
    const int page = __builtin_amdgcn_readfirstlane(bt[p]);
    const bool ok = kv4_page_ok(page, c.n_pages);
    pg.load(c.pool + ((int64_t)(ok ? page : 0) * c.Hkv + h) * kv4_slab_bytes(HD), lane);
    if (!ok) {
        pg.ks = 0xffffffffu;
#pragma unroll
        for (int x = 0; x < HD / 64; ++x) pg.vs[x] = u32x4{0u, 0u, 0u, 0u};
    }
}
// bits of a NaN in both halves of a word, of either type
#define KV4_NAN2 0x7fff7fffu

// NaN into the rows of columns [c0, c1) of a sequence and key head
template <int HD> __device__ void kv4_fill_columns(const Kv4Attn& a, const Kv4Seq& s, int h, int c0, int c1, int tid, int threads) {
    for (int i = tid; i < (c1 - c0) * (HD / 8); i += threads) {
        const int col = c0 + i / (HD / 8), j = col / a.group, head = h * a.group + col % a.group;
        const u32x4 w = {KV4_NAN2, KV4_NAN2, KV4_NAN2, KV4_NAN2};
        *reinterpret_cast<u32x4*>(a.out + (int64_t)(s.start + j) * a.out_stride + head * HD + i % (HD / 8) * 8) = w;
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Few columns: one workgroup per (chunk, tile of 16 columns and key head, sequence).
// ------------------------------------------------------------------------------------------------------------------
template <int HD, bool F16>
__global__ __launch_bounds__(256) void kv4_attn_few_kernel(Kv4View c, Kv4Rows b, Kv4Attn a) {
    __shared__ float sm[4][2][16];
    __shared__ __attribute__((aligned(16))) float so[4][16][HD + 4];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.y % c.Hkv, tile = blockIdx.y / c.Hkv, chunk = blockIdx.x, H = c.Hkv * a.group;
    const Kv4Seq s = kv4_seq_of(b, c, blockIdx.z);
    const int rows = s.n < b.max_rows ? s.n : b.max_rows;
    const int cols = rows * a.group;
    if (s.state == 1 || cols > KV4_FEW_COLUMNS || tile * 16 >= cols) return;
    const int c1 = cols < tile * 16 + 16 ? cols : tile * 16 + 16;
    if (s.state == 2) {
        if (chunk == 0) kv4_fill_columns<HD>(a, s, h, tile * 16, c1, tid, 256);
        return;
    }
    const int chunks = kv4_chunks(s.ctx), per = kv4_chunk_pages(s.ctx);
    if (chunk >= (chunks > 0 ? chunks : 1)) return;

    const int col = tile * 16 + (lane & 15), j = col / a.group, head = h * a.group + col % a.group;
    const int sees = col < cols ? s.ctx - s.n + j + 1 : 0;        // entries that this lane's column sees, may be <= 0
    const int least = s.ctx - s.n + (tile * 16) / a.group + 1;    // what the tile's first row sees
    Kv4Query<HD, F16> q[1];
    q[0].load(col < cols ? a.q + (int64_t)(s.start + j) * a.q_stride + head * HD : nullptr, lane);
    Kv4State<HD, 1> st;
    st.clear();

    const int p0 = chunk * per, pages = (s.ctx + KV4_PAGE - 1) / KV4_PAGE, p1 = pages < p0 + per ? pages : p0 + per;
    const int32_t* bt = c.table + (int64_t)s.stream * c.max_pages;
    for (int p = p0 + w; p < p1; p += 4) {
        Kv4Page<HD> pg;
        kv4_fetch<HD>(pg, c, bt, p, h, lane);
        const int first = p * KV4_PAGE, seen[1] = {sees - first};
        if (least >= first + KV4_PAGE) kv4_page_step<HD, F16, 1, false>(pg, q, st, seen, KV4_PAGE, a.c, lane);
        else kv4_page_step<HD, F16, 1, true>(pg, q, st, seen, s.ctx - first, a.c, lane);
    }
    float l = st.l[0];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
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
    // the four waves in order; a thread 8 dims of a column
    for (int i = tid; i < 16 * (HD / 8); i += 256) {
        const int k = i / (HD / 8), d = i % (HD / 8) * 8, kcol = tile * 16 + k;
        if (kcol >= c1) continue;
        float M = sm[0][0][k];
#pragma unroll
        for (int x = 1; x < 4; ++x) M = fmaxf(M, sm[x][0][k]);
        float L = 0.f, o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const float f = __builtin_amdgcn_exp2f(sm[x][0][k] - M);
            L = fmaf(sm[x][1][k], f, L);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = fmaf(so[x][k][d + e], f, o[e]);
        }
        if (chunks > 1) {
            float* sp = a.states + kv4_state_at<HD>(a, c.Hkv, blockIdx.z, h, tile, chunk);
            if (d == 0) { sp[k] = M; sp[16 + k] = L; }
#pragma unroll
            for (int e = 0; e < 8; e += 4)
                *reinterpret_cast<f32x4*>(sp + 32 + k * HD + d + e) = f32x4{o[e], o[e + 1], o[e + 2], o[e + 3]};
        } else {
            const int jj = kcol / a.group, hh = h * a.group + kcol % a.group;
            const float inv = L == 0.f ? 0.f : 1.0f / L;          // nothing seen: 0 (a NaN stays one)
            const u32x4 r = {kv4_pack2<F16>(o[0] * inv, o[1] * inv), kv4_pack2<F16>(o[2] * inv, o[3] * inv),
                             kv4_pack2<F16>(o[4] * inv, o[5] * inv), kv4_pack2<F16>(o[6] * inv, o[7] * inv)};
            *reinterpret_cast<u32x4*>(a.out + (int64_t)(s.start + jj) * a.out_stride + hh * HD + d) = r;
            if (a.norm && d == 0) a.norm[(int64_t)(s.start + jj) * H + hh] = f32x2{M, inv};
        }
    }
}

// joins the chunks of a (sequence, key head, tile) in order; a thread 4 dims of a column
template <int HD, bool F16>
__global__ __launch_bounds__(256) void kv4_attn_join_kernel(Kv4View c, Kv4Rows b, Kv4Attn a) {
    const int h = blockIdx.x % c.Hkv, tile = blockIdx.x / c.Hkv, H = c.Hkv * a.group;
    const Kv4Seq s = kv4_seq_of(b, c, blockIdx.y);
    const int rows = s.n < b.max_rows ? s.n : b.max_rows, cols = rows * a.group;
    if (s.state || cols > KV4_FEW_COLUMNS || tile * 16 >= cols) return;
    const int chunks = kv4_chunks(s.ctx);
    if (chunks <= 1) return;
    const float* sp = a.states + kv4_state_at<HD>(a, c.Hkv, blockIdx.y, h, tile, 0);
    constexpr int step = 16 * (HD + 2);
    for (int i = threadIdx.x; i < 16 * (HD / 4); i += 256) {
        const int k = i / (HD / 4), d = i % (HD / 4) * 4, col = tile * 16 + k;
        if (col >= cols) continue;
        float M = sp[k];
        for (int x = 1; x < chunks; ++x) M = fmaxf(M, sp[(int64_t)x * step + k]);
        float L = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        for (int x = 0; x < chunks; ++x) {
            const float* p = sp + (int64_t)x * step;
            const float f = __builtin_amdgcn_exp2f(p[k] - M);
            L = fmaf(p[16 + k], f, L);
            const f32x4 v = *reinterpret_cast<const f32x4*>(p + 32 + k * HD + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(v[e], f, o[e]);
        }
        const int j = col / a.group, head = h * a.group + col % a.group;
        const float inv = L == 0.f ? 0.f : 1.0f / L;
        const u32x2 r = {kv4_pack2<F16>(o[0] * inv, o[1] * inv), kv4_pack2<F16>(o[2] * inv, o[3] * inv)};
        *reinterpret_cast<u32x2*>(a.out + (int64_t)(s.start + j) * a.out_stride + head * HD + d) = r;
        if (a.norm && d == 0) a.norm[(int64_t)(s.start + j) * H + head] = f32x2{M, inv};
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Many columns (prompts): one wave per NC tiles of 16 columns and key head, the whole cache up to what its last row sees.
// ------------------------------------------------------------------------------------------------------------------
template <int HD, bool F16, int NC>
__global__ __launch_bounds__(256) void kv4_attn_many_kernel(Kv4View c, Kv4Rows b, Kv4Attn a) {
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.y, H = c.Hkv * a.group;
    const Kv4Seq s = kv4_seq_of(b, c, blockIdx.z);
    const int rows = s.n < b.max_rows ? s.n : b.max_rows, cols = rows * a.group;
    if (s.state == 1 || cols <= KV4_FEW_COLUMNS) return;
    const int c0 = (blockIdx.x * 4 + w) * (16 * NC);
    if (c0 >= cols) return;                                       // no barrier below: waves are on their own
    const int c1 = cols < c0 + 16 * NC ? cols : c0 + 16 * NC;
    if (s.state == 2) { kv4_fill_columns<HD>(a, s, h, c0, c1, lane, 64); return; }

    Kv4Query<HD, F16> q[NC];
    int sees[NC], seen[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int col = c0 + 16 * n + (lane & 15), j = col / a.group;
        q[n].load(col < c1 ? a.q + (int64_t)(s.start + j) * a.q_stride + (h * a.group + col % a.group) * HD : nullptr, lane);
        sees[n] = col < c1 ? s.ctx - s.n + j + 1 : 0;
    }
    const int least = s.ctx - s.n + c0 / a.group + 1, most = s.ctx - s.n + (c1 - 1) / a.group + 1;   // first and last row of the wave
    Kv4State<HD, NC> st;
    st.clear();
    const int32_t* bt = c.table + (int64_t)s.stream * c.max_pages;
    for (int first = 0; first < most; first += KV4_PAGE) {
        Kv4Page<HD> pg;
        kv4_fetch<HD>(pg, c, bt, first / KV4_PAGE, h, lane);
#pragma unroll
        for (int n = 0; n < NC; ++n) seen[n] = sees[n] - first;
        if (least >= first + KV4_PAGE) kv4_page_step<HD, F16, NC, false>(pg, q, st, seen, KV4_PAGE, a.c, lane);
        else kv4_page_step<HD, F16, NC, true>(pg, q, st, seen, s.ctx - first, a.c, lane);
    }
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int col = c0 + 16 * n + (lane & 15), j = col / a.group, head = h * a.group + col % a.group, g = lane >> 4;
        float l = st.l[n];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (col >= c1) continue;
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        uint16_t* op = a.out + (int64_t)(s.start + j) * a.out_stride + head * HD + 16 * g;
#pragma unroll
        for (int x = 0; x < HD / 64; ++x)
#pragma unroll
            for (int jj = 0; jj < 4; jj += 2) {
                const f32x4 (&o)[4] = st.o[n][x];
                const u32x4 r = {kv4_pack2<F16>(o[0][jj] * inv, o[1][jj] * inv), kv4_pack2<F16>(o[2][jj] * inv, o[3][jj] * inv),
                                 kv4_pack2<F16>(o[0][jj + 1] * inv, o[1][jj + 1] * inv), kv4_pack2<F16>(o[2][jj + 1] * inv, o[3][jj + 1] * inv)};
                *reinterpret_cast<u32x4*>(op + 64 * x + 4 * jj) = r;
            }
        if (a.norm && g == 0) a.norm[(int64_t)(s.start + j) * H + head] = f32x2{st.m[n], inv};
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Weights: W[stream][key head][t] += sum over the sequence's columns of exp2(s c - m) / l.  One wave per (page, key head, stream)
// forms the scores again from K (half a page's bytes, mostly still on the chip) and walks the columns in order, so no atomics.
// A stream that occurs in several sequences of the call is done, in their order, by the waves of the first of them.
// ------------------------------------------------------------------------------------------------------------------
template <int HD, bool F16>
__global__ __launch_bounds__(256) void kv4_weights_kernel(Kv4View c, Kv4Rows b, Kv4Attn a, float* weights, int64_t weights_stride) {
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.y, H = c.Hkv * a.group, seq = blockIdx.z, p = blockIdx.x * 4 + w, first = p * KV4_PAGE;
    const int stream = b.stream[seq];
    if (stream < 0 || stream >= c.n_streams) return;
    for (int i = lane; i - lane < seq; i += 64)
        if (__any(i < seq && b.stream[i < seq ? i : 0] == stream)) return;      // an earlier sequence's waves do it
    const int32_t* bt = c.table + (int64_t)stream * c.max_pages;
    Kv4Page<HD> pg;
    bool have = false;
    float sum[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) sum[e] = 0.f;
    // the sequences of this stream from here on, found 64 at a time
    uint64_t todo = 0;
    for (int i0 = seq - 64, i; ; ) {
        while (todo == 0) {
            i0 += 64;
            if (i0 >= b.n_seqs) break;
            todo = __ballot(i0 + lane < b.n_seqs && b.stream[i0 + lane < b.n_seqs ? i0 + lane : seq] == stream);
        }
        if (todo == 0) break;
        i = i0 + __builtin_ctzll(todo);
        todo &= todo - 1;
        const Kv4Seq s = kv4_seq_of(b, c, i);
        if (s.state || first >= s.ctx) continue;
        if (!have) {
            kv4_fetch<HD>(pg, c, bt, p, h, lane);
            have = true;
        }
        const int rows = s.n < b.max_rows ? s.n : b.max_rows, cols = rows * a.group;
        // rows before the first that sees this page add nothing
        int j0 = first - (s.ctx - s.n);
        j0 = j0 < 0 ? 0 : j0;
        for (int c0 = j0 * a.group / 16 * 16; c0 < cols; c0 += 16) {
            const int col = c0 + (lane & 15), j = col / a.group, head = h * a.group + col % a.group;
            Kv4Query<HD, F16> q[1];
            q[0].load(col < cols ? a.q + (int64_t)(s.start + j) * a.q_stride + head * HD : nullptr, lane);
            f32x2 norm = {0.f, 0.f};
            if (col < cols) norm = a.norm[(int64_t)(s.start + j) * H + head];
            const int seen = col < cols ? s.ctx - s.n + j + 1 - first : 0;
            f32x4 sc[1][4];
            kv4_scores<HD, F16, 1>(pg, q, sc);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float v = __builtin_amdgcn_exp2f(fmaf(sc[0][e & 3][e >> 2], a.c, -norm[0]));
                sum[e] += 16 * (lane >> 4) + e < seen ? v * norm[1] : 0.f;
            }
        }
    }
    if (!have) return;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        sum[e] += __shfl_xor(sum[e], 1);
        sum[e] += __shfl_xor(sum[e], 2);
        sum[e] += __shfl_xor(sum[e], 4);
        sum[e] += __shfl_xor(sum[e], 8);
    }
    // lane r of the group keeps token 16 g + r
    float mine = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) mine = (lane & 15) == e ? sum[e] : mine;
    const int64_t t = first + lane;
    if (t < weights_stride) {
        float* wp = weights + ((int64_t)stream * c.Hkv + h) * weights_stride + t;
        if (mine != 0.f) *wp += mine;
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Entry points
// ------------------------------------------------------------------------------------------------------------------
static int64_t states_bytes(const t3_kv4_cache* c, const t3_kv4_batch* b, int H, int* tiles, int* chunks) {
    const int64_t cols = (int64_t)b->max_rows * (H / c->Hkv), few = cols < KV4_FEW_COLUMNS ? cols : KV4_FEW_COLUMNS;
    const int64_t cap = (int64_t)c->max_pages * KV4_PAGE;
    *tiles = (int)((few + 15) / 16);
    *chunks = kv4_max_chunks((int)(b->max_ctx < cap ? b->max_ctx : cap));
    return *chunks > 1 ? (int64_t)b->n_seqs * c->Hkv * *tiles * *chunks * (16 * (c->hd + 2)) * 4 : 0;
}
static int check_heads(const t3_kv4_cache* c, int H) {
    T3_REQUIRE(H >= c->Hkv && H % c->Hkv == 0 && H / c->Hkv <= 64, "attn_kv4: query heads must be 1..64 times the key heads");
    return 0;
}

extern "C" int64_t t3_op_attn_kv4_work_bytes(const t3_kv4_cache* cache, const t3_kv4_batch* batch, int32_t H, int32_t with_weights) {
    if (kv4_check_cache(cache, 0, 1, nullptr) || kv4_check_batch(batch) || check_heads(cache, H)) return -1;
    int tiles, chunks;
    return states_bytes(cache, batch, H, &tiles, &chunks) + (with_weights ? ((int64_t)batch->rows * H * 8 + 15) / 16 * 16 : 0);
}

template <int HD, bool F16>
static int launch_attn(const Kv4View& c, const Kv4Rows& b, const Kv4Attn& a, float* weights, int64_t weights_stride, hipStream_t st) {
    constexpr int NC = 4;
    const int64_t cols = (int64_t)b.max_rows * a.group;
    T3_LAUNCH((kv4_attn_few_kernel<HD, F16>), dim3(a.chunks, a.tiles * c.Hkv, b.n_seqs), dim3(256), 0, st, c, b, a);
    if (a.chunks > 1)
        T3_LAUNCH((kv4_attn_join_kernel<HD, F16>), dim3(a.tiles * c.Hkv, b.n_seqs), dim3(256), 0, st, c, b, a);
    if (cols > KV4_FEW_COLUMNS)
        T3_LAUNCH((kv4_attn_many_kernel<HD, F16, NC>), dim3((unsigned)((cols + 64 * NC - 1) / (64 * NC)), c.Hkv, b.n_seqs), dim3(256), 0, st, c, b, a);
    if (weights) {
        const int64_t cap = (int64_t)c.max_pages * KV4_PAGE, most = b.max_ctx < cap ? b.max_ctx : cap;
        T3_LAUNCH((kv4_weights_kernel<HD, F16>), dim3((unsigned)((most + 4 * KV4_PAGE - 1) / (4 * KV4_PAGE)), c.Hkv, b.n_seqs), dim3(256), 0, st,
                  c, b, a, weights, weights_stride);
    }
    T3_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int t3_op_attn_kv4(const t3_kv4_cache* cache, const t3_kv4_batch* batch, const void* q_dev, int64_t q_stride,
                              void* out_dev, int64_t out_stride, int32_t H, int32_t dtype, float scale, float* weights_dev,
                              int64_t weights_stride, void* work_dev, int64_t work_bytes, int32_t layer, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (kv4_check_cache(cache, layer, 1, st) || kv4_check_batch(batch) || check_heads(cache, H)) return 1;
    T3_REQUIRE(q_dev && out_dev, "attn_kv4: null argument");
    T3_REQUIRE(dtype == 0 || dtype == 1, "attn_kv4: dtype must be 0 (bf16) or 1 (fp16)");
    T3_REQUIRE(scale > 0.f && scale < 1e8f, "attn_kv4: scale must be positive");
    T3_REQUIRE((int64_t)batch->max_rows * (H / cache->Hkv) <= (1 << 30), "attn_kv4: more than 2^30 rows x query heads of a key head");
    const int64_t width = (int64_t)H * cache->hd;
    T3_REQUIRE(q_stride >= width && out_stride >= width && q_stride % 8 == 0 && out_stride % 8 == 0 &&
               reinterpret_cast<uintptr_t>(q_dev) % 16 == 0 && reinterpret_cast<uintptr_t>(out_dev) % 16 == 0,
               "attn_kv4: rows must be 16-byte aligned and must not overlap");
    T3_REQUIRE(!weights_dev || weights_stride >= batch->max_ctx, "attn_kv4: weights_stride must be at least max_ctx");
    const int64_t needed = t3_op_attn_kv4_work_bytes(cache, batch, H, weights_dev != nullptr);
    T3_REQUIRE(needed == 0 || (work_dev && work_bytes >= needed && reinterpret_cast<uintptr_t>(work_dev) % 16 == 0),
               "attn_kv4: the work buffer is too small or not 16-byte aligned");
    Kv4Attn a{};
    a.q = static_cast<const uint16_t*>(q_dev); a.q_stride = q_stride;
    a.out = static_cast<uint16_t*>(out_dev); a.out_stride = out_stride;
    a.group = H / cache->Hkv;
    a.c = scale * 1.44269504088896340736f;
    const int64_t sb = states_bytes(cache, batch, H, &a.tiles, &a.chunks);
    a.states = static_cast<float*>(work_dev);
    a.norm = weights_dev ? reinterpret_cast<f32x2*>(static_cast<uint8_t*>(work_dev) + sb) : nullptr;
    const Kv4View c = kv4_view(cache, layer);
    const Kv4Rows b = kv4_rows(batch);
    if (cache->hd == 64) return dtype ? launch_attn<64, true>(c, b, a, weights_dev, weights_stride, st) : launch_attn<64, false>(c, b, a, weights_dev, weights_stride, st);
    return dtype ? launch_attn<128, true>(c, b, a, weights_dev, weights_stride, st) : launch_attn<128, false>(c, b, a, weights_dev, weights_stride, st);
}
