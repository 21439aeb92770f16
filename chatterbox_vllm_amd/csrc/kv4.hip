// 4-bit KV cache: append (quantise and write rows), read (rows back as values), eviction by accumulated attention weight, and
// the checks that every entry point of the cache shares.  Byte order: kv4_layout.h; attention: kv4_attn.hip.
#include "kv4_common.h"

// ------------------------------------------------------------------------------------------------------------------
// Append.  For each row, key head and block of 32 dims, with a = max |x|:
//   2^e = the smallest power of two with a / 2^e < 7,   code = e2m1 value nearest to x / 2^e (ties to the even code).
// A thread takes 8 dims of K and the same of V (two 16-byte loads).  The bits of |x| of either type order like the values, so the
// maxima run on 16-bit halves, K's in the low one and V's in the high one after the first step; the conversion rounds, scales and packs
// two values at a time from the type that they come in.  Bound by what it reads: 12 x 1000 rows x 8 heads of 128, 49 MB in and 13 MB
// out, 11 us (5.6 TB/s; with values widened to fp32, one wave a page and two-byte stores of V 20).  A row for each of 64 streams x 16
// heads of 64: 3.5 us, all of it launch and latency.
// ------------------------------------------------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(2))) uint16_t u16x2;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
__device__ __forceinline__ unsigned kv4_max2(unsigned a, unsigned b) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// largest |x| of eight values, in both halves' maxima
__device__ __forceinline__ unsigned kv4_absmax2(u32x4 x) {
    const unsigned m = 0x7fff7fffu;
    return kv4_max2(kv4_max2(x[0] & m, x[1] & m), kv4_max2(x[2] & m, x[3] & m));
}
template <int CTRL> __device__ __forceinline__ unsigned kv4_lane_max2(unsigned v) {
    return kv4_max2(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true));
}
template <bool F16> __device__ __forceinline__ float kv4_magnitude(unsigned half) {
    if constexpr (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)half);
    else return __uint_as_float(half << 16);
}
template <bool F16> __device__ __forceinline__ unsigned kv4_codes8(u32x4 x, float scale) {
    const unsigned w0 = x[0], w1 = x[1], w2 = x[2], w3 = x[3];
    unsigned r = 0;
#define KV4_CODES2(i)                                                                                                        \
    if constexpr (F16) r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, w##i), scale, i);           \
    else r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w##i), scale, i);
    KV4_CODES2(0) KV4_CODES2(1) KV4_CODES2(2) KV4_CODES2(3)
#undef KV4_CODES2
    return r;
}

// A workgroup takes the rows of one page: of a key head, 16 tokens a wave (PAGES), or of four heads, one a wave, where the sequences
// have too few rows to fill a page.  Rows that fill it build its slab in shared memory, which leaves in 16-byte stores; others are
// stored from where they are, two bytes of V at a time, since their neighbours may be someone else's.
struct Kv4Slice { int64_t first, slot; int lo, hi, page; };      // slot of row 0; of token 0; tokens [lo, hi) are rows; page id

__device__ __forceinline__ int kv4_slices(int n) { return (int)(((int64_t)n + KV4_PAGE - 2) / KV4_PAGE) + 1; }
__device__ __forceinline__ Kv4Slice kv4_slice(const Kv4View& c, const Kv4Seq& s, int n, int64_t x) {
    Kv4Slice r;
    r.first = (int64_t)s.ctx - s.n;
    r.slot = ((r.first >> 6) + x) * KV4_PAGE;
    const int64_t lo = r.first - r.slot, hi = r.first + n - r.slot;
    r.lo = lo > 0 ? (int)lo : 0;
    r.hi = hi < KV4_PAGE ? (int)hi : KV4_PAGE;                   // not above lo: no row of the sequence
    r.page = r.slot >= 0 && r.lo < r.hi && s.state == 0 ? c.table[(int64_t)s.stream * c.max_pages + r.slot / KV4_PAGE] : -1;
    return r;
}

template <int HD, bool F16> struct Kv4AppendItem {               // 8 dims of one row and head
    u32x4 k, v;
    __device__ __forceinline__ void load(const uint16_t* kp, const uint16_t* vp, bool in) {
        k = v = u32x4{0u, 0u, 0u, 0u};
        if (in) { k = *reinterpret_cast<const u32x4*>(kp); v = *reinterpret_cast<const u32x4*>(vp); }
    }
    // (all lanes of the row and head: the maxima are taken over every one)
    template <typename P> __device__ __forceinline__ void store(P slab, int t, int ch, bool in) const {
        const unsigned km = kv4_absmax2(k), vm = kv4_absmax2(v);
        unsigned m = kv4_max2(km & 0xffffu | vm << 16, km >> 16 | vm & 0xffff0000u);
        m = kv4_lane_max2<0x4e>(kv4_lane_max2<0xb1>(m));         // over the block of 32: neighbours, then pairs (quad_perm)
        unsigned any = kv4_lane_max2<0x141>(m);                  // over the entry: the other quad (row_half_mirror)
        if constexpr (HD == 128) any = kv4_lane_max2<0x140>(any);   // and the other eight (row_mirror)
        constexpr unsigned inf = F16 ? 0x7c00u : 0x7f80u;
        const bool bad = (any & 0xffffu) >= inf || any >> 16 >= inf;   // a NaN or an infinity somewhere in the entry
        if (!in) return;
        const int kb = kv4_scale_byte(__float_as_uint(kv4_magnitude<F16>(m & 0xffffu)));
        const int vb = kv4_scale_byte(__float_as_uint(kv4_magnitude<F16>(m >> 16)));
        const unsigned keep = bad ? 0u : ~0u, kc = kv4_codes8<F16>(k, kv4_scale(kb)) & keep, vc = kv4_codes8<F16>(v, kv4_scale(vb)) & keep;
        *reinterpret_cast<unsigned*>(slab + kv4_k_at(HD, t, ch)) = kc;
        *reinterpret_cast<uint16_t*>(slab + kv4_v_at(HD, t, ch)) = (uint16_t)vc;
        *reinterpret_cast<uint16_t*>(slab + kv4_v_at(HD, t, ch + 4)) = (uint16_t)(vc >> 16);
        if (ch % KV4_BLOCK == 0) {
            slab[kv4_ks_at(HD, t, ch)] = (uint8_t)(bad ? KV4_NAN_SCALE : kb);
            slab[kv4_vs_at(HD, t, ch)] = (uint8_t)(bad ? KV4_MIN_SCALE : vb);
        }
    }
};

template <int HD, bool F16, bool PAGES>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4View c, Kv4Rows b, const uint16_t* __restrict__ k,
                                                         const uint16_t* __restrict__ v, int64_t k_stride, int64_t v_stride) {
    constexpr int T = HD / 8, STEP = 64 / T, SLAB = KV4_PAGE * (HD + HD / 16);   // lanes of a row, rows a step
    constexpr int HEADS = PAGES ? 1 : 4, PART = KV4_PAGE / (4 / HEADS);          // heads of a workgroup, tokens of a wave
    const Kv4Seq s = kv4_seq_of(b, c, blockIdx.y);
    if (s.state) return;
    const int n = s.n < b.max_rows ? s.n : b.max_rows, lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ch = lane % T * 8, groups = (c.Hkv + HEADS - 1) / HEADS, x0 = blockIdx.x / groups, slices = kv4_slices(n);
    const int h = (blockIdx.x - x0 * groups) * HEADS + (PAGES ? 0 : w), first = PAGES ? w * PART : 0;
    if (h >= c.Hkv) return;
    for (int64_t x = x0; x < slices; x += gridDim.x / groups) {
        const Kv4Slice r = kv4_slice(c, s, n, x);
        if (!kv4_page_ok(r.page, c.n_pages)) continue;
        const int64_t row = s.start + r.slot - r.first;          // of token 0
        const uint16_t* kp = k + row * k_stride + h * HD + ch;
        const uint16_t* vp = v + row * v_stride + h * HD + ch;
        uint8_t* slab = c.pool + ((int64_t)r.page * c.Hkv + h) * SLAB;
        if constexpr (PAGES) {
            if (r.lo == 0 && r.hi == KV4_PAGE) {
                __shared__ __attribute__((aligned(16))) uint8_t built[SLAB];
                Kv4AppendItem<HD, F16> a[PART / STEP];
#pragma unroll
                for (int j = 0; j < PART / STEP; ++j) {
                    const int t = first + j * STEP + lane / T;
                    a[j].load(kp + t * k_stride, vp + t * v_stride, true);
                }
#pragma unroll
                for (int j = 0; j < PART / STEP; ++j) a[j].store(built, first + j * STEP + lane / T, ch, true);
                __syncthreads();
                for (int q = threadIdx.x; q < SLAB / 16; q += 256) reinterpret_cast<u32x4*>(slab)[q] = reinterpret_cast<const u32x4*>(built)[q];
                __syncthreads();
                continue;
            }
        }
        const int hi = r.hi < first + PART ? r.hi : first + PART;
        for (int t0 = r.lo > first ? r.lo : first; t0 < hi; t0 += STEP) {
            const int t = t0 + lane / T;
            Kv4AppendItem<HD, F16> a;
            a.load(kp + t * k_stride, vp + t * v_stride, t < hi);
            a.store(slab, t, ch, t < hi);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Read: the inverse, a thread 8 dims of K and of V.  Bound by what it writes: 8 streams x 30 layers x 16 heads x 640 entries of 64, 167 MB
// in and 629 MB out, 133 us (6.0 TB/s; straight from memory with divisions per thread 268).
// ------------------------------------------------------------------------------------------------------------------
template <bool F16> __device__ __forceinline__ u32x4 kv4_values8(unsigned codes, unsigned byte, bool nan) {
    if constexpr (F16) {
        // from 57344 on a value appended from fp16 is held as 4 * 2^14, and bf16 has larger ones: cut at the type's largest instead of
        // becoming infinite
        const f16x2 most = {(_Float16)65504.f, (_Float16)65504.f};
        const float sc = kv4_scale(byte);
        const f16x2 p[4] = {__builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, sc, 0)),
                            __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, sc, 1)),
                            __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, sc, 2)),
                            __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, sc, 3))};
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            o[i] = nan ? 0x7fff7fffu : __builtin_bit_cast(unsigned, __builtin_elementwise_min(__builtin_elementwise_max(p[i], -most), most));
        return o;
    } else {
        const float sc = nan ? __uint_as_float(0x7f800000u) : kv4_scale(byte);
        return u32x4{kv4_pair<0>(codes, sc), kv4_pair<1>(codes, sc), kv4_pair<2>(codes, sc), kv4_pair<3>(codes, sc)};
    }
}

// The slab comes in through shared memory, 16 bytes a lane.  A workgroup takes a page of four heads at head_dim 64, one a wave, and of
// one head at 128 (64 x 100 rows x 16 heads of 64: 7.8 us, by one head 9.1; 64 x 33 rows x 8 heads of 128: 6.0 and 5.3).
template <int HD, bool F16>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4View c, Kv4Rows b, int64_t layer_stride, uint16_t* __restrict__ k,
                                                       uint16_t* __restrict__ v) {
    constexpr bool PAGES = HD == 128;
    constexpr int T = HD / 8, SLAB = KV4_PAGE * (HD + HD / 16), HEADS = PAGES ? 1 : 4, LANES = 256 / HEADS, STEP = LANES / T;
    constexpr int UNITS = SLAB / 16, EACH = (UNITS + LANES - 1) / LANES;
    __shared__ __attribute__((aligned(16))) uint8_t slabs[HEADS][SLAB];
    const Kv4Seq s = kv4_seq_of(b, c, blockIdx.y);
    if (s.state == 1) return;
    const uint8_t* pool = c.pool + (int64_t)blockIdx.z * layer_stride;
    const int n = s.n < b.max_rows ? s.n : b.max_rows, w = __builtin_amdgcn_readfirstlane(threadIdx.x / LANES), lane = threadIdx.x % LANES;
    const int ch = lane % T * 8, groups = (c.Hkv + HEADS - 1) / HEADS, x0 = blockIdx.x / groups, slices = kv4_slices(n);
    const int h = (blockIdx.x - x0 * groups) * HEADS + w;
    if (h >= c.Hkv) return;
    u32x4* slab = reinterpret_cast<u32x4*>(slabs[w]);
    const auto wait = [] {
        if constexpr (PAGES) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    for (int64_t x = x0; x < slices; x += gridDim.x / groups) {
        const Kv4Slice r = kv4_slice(c, s, n, x);
        const bool ok = kv4_page_ok(r.page, c.n_pages), none = s.state == 0 && r.slot < 0;   // none: entries before the first
        if (ok) {
            const u32x4* from = reinterpret_cast<const u32x4*>(pool + ((int64_t)r.page * c.Hkv + h) * SLAB);
            u32x4 in[EACH];
#pragma unroll
            for (int q = 0; q < EACH; ++q)
                if (q * LANES + lane < UNITS) in[q] = from[q * LANES + lane];
#pragma unroll
            for (int q = 0; q < EACH; ++q)
                if (q * LANES + lane < UNITS) slab[q * LANES + lane] = in[q];
            wait();
        }
        const int64_t at = (((int64_t)blockIdx.z * b.rows + s.start + r.slot - r.first) * c.Hkv + h) * HD + ch;
        for (int t = r.lo + lane / T; t < r.hi; t += STEP) {
            u32x4 ko = {0u, 0u, 0u, 0u}, vo = ko;
            if (ok) {
                const uint8_t* p = slabs[w];
                const unsigned kc = *reinterpret_cast<const unsigned*>(p + kv4_k_at(HD, t, ch));
                const unsigned vc = *reinterpret_cast<const uint16_t*>(p + kv4_v_at(HD, t, ch)) |
                                    (unsigned)*reinterpret_cast<const uint16_t*>(p + kv4_v_at(HD, t, ch + 4)) << 16;
                const unsigned kb = p[kv4_ks_at(HD, t, ch)], vb = p[kv4_vs_at(HD, t, ch)];
                ko = kv4_values8<F16>(kc, kb, kb == KV4_NAN_SCALE);
                vo = kv4_values8<F16>(vc, vb, kb == KV4_NAN_SCALE);
            } else if (!none) {
                ko = kv4_values8<F16>(0u, 0u, true);
                vo = ko;
            }
            *reinterpret_cast<u32x4*>(k + at + (int64_t)t * c.Hkv * HD) = ko;
            *reinterpret_cast<u32x4*>(v + at + (int64_t)t * c.Hkv * HD) = vo;
        }
        if (ok) wait();
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Eviction.  Of an entry's ctx tokens [0, sink) and [ctx - recent, ctx) stay; of the others the `need` largest weights, ties to
// the lower index, so that the set is what any correct sort would give.  Per (entry, key head, layer) on its own:
//   T = the largest key with at least `need` candidate keys >= T, found from the highest bit in which they differ down;
//   what is above T stays, and the first need - |above T| of those equal to it.
// Bound by the bytes moved: the kept entries lie scattered, so every line of the source is read (8 streams x 30 layers x 16 heads of
// 64, 1500..2011 entries to 640: 457 MB, with 208 MB written 690 MB in 172 us, 4.0 TB/s; choice and move as two launches 355).  One layer
// of 4 streams x 16 heads is latency, a chain of about eight loads and barriers: 9 us (17.4).
// ------------------------------------------------------------------------------------------------------------------
struct Kv4Evict {
    const int32_t* src; const int32_t* dst; const int32_t* ctx;
    float* weights; int64_t weights_stride;
    int32_t* new_ctx; int32_t* kept;
    int n, max_ctx, keep, sink, recent;
};
struct Kv4Entry { int src, dst, ctx; bool ok; };

// the entry's numbers; not ok: they fit neither the cache nor the call
__device__ __forceinline__ Kv4Entry kv4_entry(const Kv4View& c, const Kv4Evict& e, int i) {
    Kv4Entry x{e.src[i], e.dst[i], e.ctx[i], true};
    x.ok = x.src >= 0 && x.src < c.n_streams && x.dst >= 0 && x.dst < c.n_streams && x.src != x.dst && x.ctx >= 0 && x.ctx <= e.max_ctx &&
           x.ctx <= (int64_t)c.max_pages * KV4_PAGE;
    return x;
}
// this thread's share of what else refuses an entry: its destination taken by an entry before it or read by any; pages (sp: of its
// source, dp: of its destination) outside the pool, or both read and written
template <int THREADS> __device__ __forceinline__ bool kv4_entry_taken(const Kv4Evict& e, const Kv4Entry& x, int i) {
    bool bad = false;
    for (int o = threadIdx.x; o < e.n; o += THREADS) bad = bad || (o < i && e.dst[o] == x.dst) || e.src[o] == x.dst;
    return bad;
}
template <int THREADS> __device__ __forceinline__ bool kv4_pages_bad(const int32_t* sp, const int32_t* dp, int ns, int nd, int n_pages) {
    const int tid = threadIdx.x;
    bool bad = false;
    for (int o = tid >> 4; o < ns; o += THREADS >> 4) {
        const int page = sp[o];
        bad = bad || !kv4_page_ok(page, n_pages);
        for (int d = tid & 15; d < nd; d += 16) bad = bad || dp[d] == page;
    }
    for (int d = tid; d < nd; d += THREADS) bad = bad || !kv4_page_ok(dp[d], n_pages);
    return bad;
}
template <int THREADS> __device__ __forceinline__ void kv4_refuse(const Kv4Evict& e, int32_t* kept, int i, bool first) {
    for (int j = threadIdx.x; j < e.keep; j += THREADS) kept[j] = -1;
    if (first && threadIdx.x == 0) e.new_ctx[i] = -1;
}
// what is behind the kept ones
template <int THREADS> __device__ __forceinline__ void kv4_clear_rest(const Kv4Evict& e, int32_t* kept, float* wd, int left) {
    for (int j = left + threadIdx.x; j < e.keep; j += THREADS) kept[j] = -1;
    for (int64_t j = left + threadIdx.x; j < e.weights_stride; j += THREADS) wd[j] = 0.f;
}

// One wave writes one page of the destination: token t becomes old[t] of the source for t < n, nothing behind.  page_of(old): the
// source's page.  K moves in pieces of one token and lane group (hd / 8 bytes), V in two bytes from each of eight tokens, whose
// addresses the lanes leave each other in `where`, scales bytewise; all of a lane's loads are in flight together.
template <int HD, typename Index, typename PageOf>
__device__ __forceinline__ void kv4_move_page(uint8_t* pool, int Hkv, int h, const Index* old, int n, int to_page, const uint8_t** where,
                                              PageOf page_of) {
    typedef typename std::conditional<HD == 64, u32x2, u32x4>::type piece_t;
    const int t = threadIdx.x & 63, t0 = t % 8 * 8, d = t / 8 * 4;
    const auto slab = [&](int page) { return pool + ((int64_t)page * Hkv + h) * kv4_slab_bytes(HD); };
    uint8_t* to = slab(to_page);
    const bool has = t < n;
    const int mine = old[has ? t : 0], at = mine % KV4_PAGE;
    const uint8_t* p = slab(page_of(mine));
    where[t] = p + kv4_v_at(HD, at, 0);
    piece_t k[4];
    uint8_t sc[HD / 16];
#pragma unroll
    for (int g = 0; g < 4; ++g) k[g] = *reinterpret_cast<const piece_t*>(p + kv4_k_at(HD, at, g * (HD / 4)));
#pragma unroll
    for (int x = 0; x < HD / 16; ++x) sc[x] = p[64 * HD + x * KV4_PAGE + at];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint16_t two[8][HD / 32];                                    // dims d + 32 x of token t0 + j
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint8_t* q = where[t0 + j] + d * 4;
#pragma unroll
        for (int x = 0; x < HD / 32; ++x) two[j][x] = *reinterpret_cast<const uint16_t*>(q + (x / 2) * 2048 + (x & 1) * 128);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) *reinterpret_cast<piece_t*>(to + kv4_k_at(HD, t, g * (HD / 4))) = has ? k[g] : piece_t{};
#pragma unroll
    for (int x = 0; x < HD / 16; ++x) to[64 * HD + x * KV4_PAGE + t] = has ? sc[x] : (uint8_t)KV4_MIN_SCALE;
    const int some = n - t0;
#pragma unroll
    for (int x = 0; x < HD / 32; ++x) {
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned both = two[2 * j][x] | (unsigned)two[2 * j + 1][x] << 16;
            v[j] = 2 * j + 1 < some ? both : 2 * j < some ? both & 0xffffu : 0u;
        }
        *reinterpret_cast<u32x4*>(to + kv4_v_at(HD, t0, d) + (x / 2) * 2048 + (x & 1) * 128) = v;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// sum over the lanes before and including this one
__device__ __forceinline__ int kv4_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);          // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);          // lane 15 of rows 0 and 2, then lane 31, to what follows
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
    return x;
}
__device__ __forceinline__ unsigned kv4_or_scan(unsigned x) {
    x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false);
    x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false);
    x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false);
    x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false);
    x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);
    x |= (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);
    return x;
}
// a barrier for shared memory alone: stores to global memory stay in flight
__device__ __forceinline__ void kv4_lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Entries of at most THREADS * PER tokens, with MOVE choice and move in one launch.  The weights go through shared memory to threads that have
// PER neighbouring ones.  The bits that all candidates share are skipped; a histogram of the next 8 gives the bin of T, and so on
// within it, until a bin stays whole: two rounds for weights that differ, 1300 clocks each (bit by bit 15 steps of 520).  Every wave
// reads the histogram for itself.
template <int HD, int THREADS, int PER, bool MOVE>
__global__ __launch_bounds__(THREADS) void kv4_evict_kernel(Kv4View c, Kv4Evict e, int64_t layer_stride) {
    constexpr int WAVES = THREADS / 64, MOST = THREADS * PER;
    __shared__ __attribute__((aligned(16))) float weight[MOST];
    __shared__ uint16_t list[MOST];
    __shared__ int32_t pages[2][MOST / KV4_PAGE];                // source, destination
    __shared__ __attribute__((aligned(16))) int hist[4 * 256];   // a round each
    __shared__ const uint8_t* where[MOVE ? WAVES : 1][64];
    __shared__ unsigned differ[WAVES];
    __shared__ int ends[WAVES], refused;
    const int h = blockIdx.x, i = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    int32_t* kept = e.kept + (((int64_t)layer * e.n + i) * c.Hkv + h) * e.keep;
    const bool first = h == 0 && layer == 0;
    const Kv4Entry x = kv4_entry(c, e, i);
    const int ctx = x.ok ? x.ctx : 0, left = ctx < e.keep ? ctx : e.keep;
    const int ns = (ctx + KV4_PAGE - 1) / KV4_PAGE, nd = (left + KV4_PAGE - 1) / KV4_PAGE;
    const bool all = ctx <= e.keep;
    const int a = all ? ctx : e.sink, z = all ? ctx : ctx - e.recent, need = all ? 0 : e.keep - e.sink - e.recent;
    const int src = x.ok ? x.src : 0, dst = x.ok ? x.dst : 0;
    const float* ws = e.weights + (((int64_t)layer * c.n_streams + src) * c.Hkv + h) * e.weights_stride;
    float* wd = e.weights + (((int64_t)layer * c.n_streams + dst) * c.Hkv + h) * e.weights_stride;
    const float one = need > 0 ? ws[a] : 0.f;
    {
        float wt[PER];
#pragma unroll
        for (int p = 0; p < PER; ++p) wt[p] = tid + THREADS * p < ctx ? ws[tid + THREADS * p] : 0.f;
        if (tid < ns) pages[0][tid] = c.table[(int64_t)src * c.max_pages + tid];
        if (tid < nd) pages[1][tid] = c.table[(int64_t)dst * c.max_pages + tid];
        for (int o = tid; o < 1024; o += THREADS) hist[o] = 0;
        if (tid == 0) refused = !x.ok;
#pragma unroll
        for (int p = 0; p < PER; ++p) weight[tid + THREADS * p] = wt[p];
    }
    const bool taken = kv4_entry_taken<THREADS>(e, x, i);
    __syncthreads();
    if (taken || kv4_pages_bad<THREADS>(pages[0], pages[1], ns, nd, c.n_pages)) refused = 1;

    // this thread's: tokens base .. base + PER - 1; bit p of `cand`: one to choose from
    const int base = tid * PER;
    const unsigned ref = kv4_weight_key(__float_as_uint(one));
    unsigned key[PER], cand = 0, diff = 0;
#pragma unroll
    for (int p = 0; p < PER; p += 4) {
        const f32x4 f = *reinterpret_cast<const f32x4*>(weight + base + p);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const bool in = base + p + q >= a && base + p + q < z;   // (none where nothing is to be chosen and all stay)
            key[p + q] = kv4_weight_key(__float_as_uint(f[q]));
            cand |= in ? 1u << (p + q) : 0u;
            diff |= in ? key[p + q] ^ ref : 0u;
        }
    }
    diff = kv4_or_scan(diff);
    if (lane == 63) differ[w] = diff;
    __syncthreads();
    if (refused) {
        for (int j = tid; j < e.keep; j += THREADS) kept[j] = -1;
        if (first && tid == 0) e.new_ctx[i] = -1;
        return;
    }
    diff = 0;
#pragma unroll
    for (int o = 0; o < WAVES; ++o) diff |= differ[o];

    // T, and how many of those equal to it stay
    int bits = __builtin_amdgcn_readfirstlane(diff ? 32 - __clz((int)diff) : 0), want = need;
    unsigned T = __builtin_amdgcn_readfirstlane(bits == 32 ? 0u : ref >> bits << bits);
    if (need == 0) T = ~0u;                                      // (no weight's key) none of the candidates
    else {                                                       // 0 < need < z - a
        for (int* hr = hist; bits > 0; hr += 256) {
            const int low = bits > 8 ? bits - 8 : 0;             // bits [low, bits)
            const unsigned mask = (1u << (bits - low)) - 1;
#pragma unroll
            for (int p = 0; p < PER; ++p)
                if ((cand >> p & 1u) && (bits == 32 || key[p] >> bits == T >> bits)) atomicAdd(&hr[key[p] >> low & mask], 1);
            kv4_lds_barrier();
            const int4 b4 = *reinterpret_cast<const int4*>(hr + 4 * (63 - lane));   // from the top
            const int b[4] = {b4.x, b4.y, b4.z, b4.w};
            const int sum = b[0] + b[1] + b[2] + b[3], upto = kv4_scan(sum);
            int above = upto - sum, bin = 4 * (63 - lane) + 3, here = b[3];
            const uint64_t at = __ballot(above < want && upto >= want);
#pragma unroll
            for (int o = 2; o >= 0; --o)
                if (above + here < want) { above += here; here = b[o]; bin = 4 * (63 - lane) + o; }
            const int from = __ffsll((unsigned long long)at) - 1;
            T |= (unsigned)__builtin_amdgcn_readlane(bin, from) << low;
            want -= __builtin_amdgcn_readlane(above, from);
            if (__builtin_amdgcn_readlane(here, from) == want) break;
            bits = low;
        }
    }
    // places in the order of the tokens, from the numbers of (those that stay) | (those equal to T) << 16
    unsigned stay = 0, tied = 0;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        const bool in = cand >> p & 1u;
        stay |= (in ? key[p] > T : base + p < ctx) ? 1u << p : 0u;
        tied |= in && key[p] == T ? 1u << p : 0u;
    }
    const int mine = __popc(stay) | __popc(tied) << 16, upto = kv4_scan(mine);
    if (lane == 63) ends[w] = upto;
    kv4_lds_barrier();
    int before = upto - mine;
#pragma unroll
    for (int o = 0; o < WAVES; ++o) before += o < w ? ends[o] : 0;
    int room = want - (before >> 16), out = (before & 0xffff) + (room < 0 ? want : before >> 16);
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        const bool tie = tied >> p & 1u;
        if ((stay >> p & 1u) || (tie && room > 0)) list[out++] = (uint16_t)(base + p);
        room -= tie;
    }
    kv4_lds_barrier();
    if constexpr (MOVE) {
        uint8_t* pool = c.pool + (int64_t)layer * layer_stride;
        for (int pg = w; pg < nd; pg += WAVES) {
            const int n = left - pg * KV4_PAGE;
            kv4_move_page<HD>(pool, c.Hkv, h, list + pg * KV4_PAGE, n < KV4_PAGE ? n : KV4_PAGE, pages[1][pg], where[w],
                              [&](int old) { return pages[0][old / KV4_PAGE]; });
        }
    }
    for (int j = tid; j < e.keep; j += THREADS) kept[j] = j < left ? list[j] : -1;
    for (int64_t j = tid; j < e.weights_stride; j += THREADS) wd[j] = j < left ? weight[list[j]] : 0.f;
    if (first && tid == 0) e.new_ctx[i] = left;
}

// Longer entries than a workgroup holds: the weights are read again for each of four rounds of an 8-bit radix histogram and once for
// the places.
#define KV4_CHOOSE_THREADS 1024

// sum over the workgroup's threads before this one; total in *all
__device__ __forceinline__ int kv4_prefix(int v, int* wave_sums, int* all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) { const int y = __shfl_up(x, o); if (lane >= o) x += y; }
    __syncthreads();                                             // the sums of the call before have been read
    if (lane == 63) wave_sums[w] = x;
    __syncthreads();
    int before = 0, total = 0;
    for (int i = 0; i < KV4_CHOOSE_THREADS / 64; ++i) { const int t = wave_sums[i]; before += i < w ? t : 0; total += t; }
    *all = total;
    return before + x - v;
}

// What kv4_pages_bad finds, in time that grows with the pages and not with their square: the destination's are marked in shared memory,
// KV4_MARKS page ids at a time, and the source's looked up.  (One head of 64, 2^20 entries to half of them: the whole eviction 2.7 ms, by
// pairs of pages 21; 2^22 entries 13.7 and 326.)
#define KV4_MARKS (1 << 19)
__device__ __forceinline__ bool kv4_many_pages_bad(const int32_t* sp, const int32_t* dp, int ns, int nd, int n_pages, unsigned* marks) {
    const int tid = threadIdx.x;
    bool bad = false;
    for (int o = tid; o < ns; o += KV4_CHOOSE_THREADS) bad = bad || !kv4_page_ok(sp[o], n_pages);
    for (int d = tid; d < nd; d += KV4_CHOOSE_THREADS) bad = bad || !kv4_page_ok(dp[d], n_pages);
    for (int64_t from = 0; from < n_pages; from += KV4_MARKS) {
        const int here = n_pages - from < KV4_MARKS ? (int)(n_pages - from) : KV4_MARKS;
        for (int x = tid; x < (here + 31) / 32; x += KV4_CHOOSE_THREADS) marks[x] = 0;
        __syncthreads();
        for (int d = tid; d < nd; d += KV4_CHOOSE_THREADS) {
            const int64_t at = dp[d] - from;
            if (at >= 0 && at < here) atomicOr(&marks[at >> 5], 1u << (at & 31));
        }
        __syncthreads();
        for (int o = tid; o < ns; o += KV4_CHOOSE_THREADS) {
            const int64_t at = sp[o] - from;
            if (at >= 0 && at < here) bad = bad || (marks[at >> 5] >> (at & 31) & 1u);
        }
        __syncthreads();
    }
    return bad;
}

__global__ __launch_bounds__(KV4_CHOOSE_THREADS) void kv4_choose_kernel(Kv4View c, Kv4Evict e) {
    __shared__ unsigned marks[KV4_MARKS / 32];
    __shared__ int hist[256];
    __shared__ int wave_sums[KV4_CHOOSE_THREADS / 64];
    __shared__ int pick[2];
    const int h = blockIdx.x, i = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x;
    int32_t* kept = e.kept + (((int64_t)layer * e.n + i) * c.Hkv + h) * e.keep;
    const bool first = h == 0 && layer == 0;
    const Kv4Entry x = kv4_entry(c, e, i);
    if (!x.ok) { kv4_refuse<KV4_CHOOSE_THREADS>(e, kept, i, first); return; }
    const int ctx = x.ctx, left = ctx < e.keep ? ctx : e.keep;
    const bool taken = kv4_entry_taken<KV4_CHOOSE_THREADS>(e, x, i);
    const bool bad = kv4_many_pages_bad(c.table + (int64_t)x.src * c.max_pages, c.table + (int64_t)x.dst * c.max_pages,
                                        (int)(((int64_t)ctx + KV4_PAGE - 1) / KV4_PAGE), (int)(((int64_t)left + KV4_PAGE - 1) / KV4_PAGE), c.n_pages, marks);
    if (__syncthreads_or(taken || bad)) { kv4_refuse<KV4_CHOOSE_THREADS>(e, kept, i, first); return; }
    const float* w = e.weights + (((int64_t)layer * c.n_streams + x.src) * c.Hkv + h) * e.weights_stride;
    float* wd = e.weights + (((int64_t)layer * c.n_streams + x.dst) * c.Hkv + h) * e.weights_stride;

    unsigned least = 0;                                          // the smallest key that stays
    int ties = 0;                                                // how many of that key stay
    const bool all = ctx <= e.keep;
    const int a = all ? ctx : e.sink, z = all ? ctx : ctx - e.recent, need = all ? 0 : e.keep - e.sink - e.recent;
    if (need > 0) {                                              // 0 < need < z - a
        int want = need;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int t = a + tid; t < z; t += KV4_CHOOSE_THREADS) {
                const unsigned key = kv4_weight_key(__float_as_uint(w[t]));
                if (shift == 24 || key >> (shift + 8) == least >> (shift + 8)) atomicAdd(&hist[key >> shift & 255], 1);
            }
            __syncthreads();
            // bins from the top: the bin in which the count reaches `want`
            int total;
            const int mine = tid < 256 ? hist[255 - tid] : 0;
            const int above = kv4_prefix(mine, wave_sums, &total);
            if (tid < 256 && above < want && above + mine >= want) { pick[0] = 255 - tid; pick[1] = above; }
            __syncthreads();
            least |= (unsigned)pick[0] << shift;
            want -= pick[1];
            __syncthreads();
        }
        ties = want;
    }
    // kept indices in order
    int out = 0, tied = 0;
    for (int t0 = 0; t0 < ctx; t0 += KV4_CHOOSE_THREADS) {
        const int t = t0 + tid;
        const bool in = t < ctx, sure = in && (t < a || t >= z);
        const float wt = in ? w[t] : 0.f;
        const unsigned key = kv4_weight_key(__float_as_uint(wt));
        const bool tie = in && !sure && need > 0 && key == least;
        int n_tied, n_out;
        const int tie_at = tied + kv4_prefix(tie ? 1 : 0, wave_sums, &n_tied);
        const bool stay = sure || (in && need > 0 && key > least) || (tie && tie_at < ties);
        const int at = out + kv4_prefix(stay ? 1 : 0, wave_sums, &n_out);
        if (stay) { kept[at] = t; wd[at] = wt; }
        tied += n_tied;
        out += n_out;
    }
    kv4_clear_rest<KV4_CHOOSE_THREADS>(e, kept, wd, left);
    if (first && tid == 0) e.new_ctx[i] = left;
}

template <int HD>
__global__ __launch_bounds__(256) void kv4_move_kernel(Kv4View c, Kv4Evict e, int64_t layer_stride) {
    __shared__ int lists[4][KV4_PAGE];
    __shared__ const uint8_t* where[4][KV4_PAGE];
    const int h = blockIdx.y % c.Hkv, i = blockIdx.y / c.Hkv, layer = blockIdx.z, lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pg = blockIdx.x * 4 + w;
    const int n = e.new_ctx[i] - pg * KV4_PAGE;                  // not positive for a refused entry (-1)
    const int32_t* kept = e.kept + (((int64_t)layer * e.n + i) * c.Hkv + h) * e.keep + pg * KV4_PAGE;
    if (lane < n) lists[w][lane] = kept[lane];
    __syncthreads();
    if (n <= 0) return;
    const int32_t* sp = c.table + (int64_t)e.src[i] * c.max_pages;
    kv4_move_page<HD>(c.pool + (int64_t)layer * layer_stride, c.Hkv, h, lists[w], n < KV4_PAGE ? n : KV4_PAGE,
                      c.table[(int64_t)e.dst[i] * c.max_pages + pg], where[w], [&](int old) { return sp[old / KV4_PAGE]; });
}

// ------------------------------------------------------------------------------------------------------------------
// Entry points
// ------------------------------------------------------------------------------------------------------------------
int kv4_check_cache(const t3_kv4_cache* c, int layer, int n_layers, hipStream_t st) {
    T3_REQUIRE(c && c->pool_dev && c->block_table_dev, "kv4: null argument");
    T3_REQUIRE(c->hd == 64 || c->hd == 128, "kv4: head_dim must be 64 or 128");
    T3_REQUIRE(c->Hkv >= 1 && c->Hkv <= 1024, "kv4: 1..1024 key/value heads");
    T3_REQUIRE(c->n_pages >= 1 && c->n_streams >= 1 && c->max_pages >= 1, "kv4: empty cache");
    T3_REQUIRE(c->max_pages <= (1 << 24), "kv4: more than 2^30 entries per stream");
    T3_REQUIRE(reinterpret_cast<uintptr_t>(c->pool_dev) % 16 == 0, "kv4: the pool must be 16-byte aligned");
    T3_REQUIRE(c->n_layers >= 1 && layer >= 0 && n_layers >= 1 && n_layers <= 4096 && layer <= c->n_layers - n_layers, "kv4: layer out of range");
    T3_REQUIRE(c->n_layers == 1 || (c->layer_stride % 16 == 0 &&
                                    c->layer_stride / (kv4_slab_bytes(c->hd) * (int64_t)c->Hkv) >= c->n_pages),
               "kv4: layers overlap, or the layer stride is not a multiple of 16");
    if (st) {
        hipDevice_t sdev = -1;
        int cur = -1;
        T3_HIP_CHECK(hipStreamGetDevice(st, &sdev));
        T3_HIP_CHECK(hipGetDevice(&cur));
        T3_REQUIRE((int)sdev == cur, "kv4: the stream belongs to another device than the current one");
    }
    return 0;
}
int kv4_check_batch(const t3_kv4_batch* b) {
    T3_REQUIRE(b && b->seq_start_dev && b->stream_dev && b->ctx_dev, "kv4: null argument");
    T3_REQUIRE(b->n_seqs >= 1 && b->n_seqs <= 65535, "kv4: 1..65535 sequences per call");
    T3_REQUIRE(b->rows >= 1 && b->max_rows >= 1 && b->max_rows <= b->rows && b->max_ctx >= 1, "kv4: bad bounds of the batch");
    return 0;
}

extern "C" int64_t t3_op_kv4_page_bytes(int32_t Hkv, int32_t hd) {
    return (hd == 64 || hd == 128) && Hkv >= 1 && Hkv <= 1024 ? (int64_t)Hkv * kv4_slab_bytes(hd) : 0;
}

// workgroups along the pages of a sequence, one a key head or one for four; capped (the kernels stride over the rest)
static int page_groups(const t3_kv4_cache* c, const t3_kv4_batch* b, bool pages) {
    const int64_t heads = pages ? c->Hkv : (c->Hkv + 3) / 4, slices = ((int64_t)b->max_rows + KV4_PAGE - 2) / KV4_PAGE + 1;
    return (int)(heads * (slices < 4096 ? slices : 4096));
}
template <int HD, bool F16> static void kv4_append_launch(const t3_kv4_cache* cache, const t3_kv4_batch* batch, int layer, const uint16_t* k,
                                                          const uint16_t* v, int64_t k_stride, int64_t v_stride, hipStream_t st) {
    // 64 sequences of 5 rows x 8 heads of 128: 4.4 us by pages, 3.8 by four heads; 17 rows: 5.4 and 5.6; 33: 6.6 and 8.9;
    // 12 of 1700: 18.5 and 26
    const bool pages = batch->max_rows >= 32;
    const dim3 grid(page_groups(cache, batch, pages), batch->n_seqs);
    const Kv4View c = kv4_view(cache, layer);
    const Kv4Rows b = kv4_rows(batch);
    if (pages) T3_LAUNCH((kv4_append_kernel<HD, F16, true>), grid, dim3(256), 0, st, c, b, k, v, k_stride, v_stride);
    else T3_LAUNCH((kv4_append_kernel<HD, F16, false>), grid, dim3(256), 0, st, c, b, k, v, k_stride, v_stride);
}
template <int HD, bool F16> static void kv4_read_launch(const t3_kv4_cache* cache, const t3_kv4_batch* batch, int layer, int n_layers, uint16_t* k,
                                                        uint16_t* v, hipStream_t st) {
    const dim3 grid(page_groups(cache, batch, HD == 128), batch->n_seqs, n_layers);
    T3_LAUNCH((kv4_read_kernel<HD, F16>), grid, dim3(256), 0, st, kv4_view(cache, layer), kv4_rows(batch), cache->layer_stride, k, v);
}

extern "C" int t3_op_kv4_append(const t3_kv4_cache* cache, const t3_kv4_batch* batch, const void* k_dev, const void* v_dev,
                                int64_t k_stride, int64_t v_stride, int32_t dtype, int32_t layer, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (kv4_check_cache(cache, layer, 1, st) || kv4_check_batch(batch)) return 1;
    T3_REQUIRE(k_dev && v_dev, "kv4_append: null argument");
    T3_REQUIRE(dtype == 0 || dtype == 1, "kv4_append: dtype must be 0 (bf16) or 1 (fp16)");
    const int64_t width = (int64_t)cache->Hkv * cache->hd;
    T3_REQUIRE(k_stride >= width && v_stride >= width && k_stride % 8 == 0 && v_stride % 8 == 0 &&
               reinterpret_cast<uintptr_t>(k_dev) % 16 == 0 && reinterpret_cast<uintptr_t>(v_dev) % 16 == 0,
               "kv4_append: rows must be 16-byte aligned and must not overlap");
    const uint16_t* k = static_cast<const uint16_t*>(k_dev);
    const uint16_t* v = static_cast<const uint16_t*>(v_dev);
    if (cache->hd == 64 && dtype == 0) kv4_append_launch<64, false>(cache, batch, layer, k, v, k_stride, v_stride, st);
    else if (cache->hd == 64) kv4_append_launch<64, true>(cache, batch, layer, k, v, k_stride, v_stride, st);
    else if (dtype == 0) kv4_append_launch<128, false>(cache, batch, layer, k, v, k_stride, v_stride, st);
    else kv4_append_launch<128, true>(cache, batch, layer, k, v, k_stride, v_stride, st);
    T3_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int t3_op_kv4_read(const t3_kv4_cache* cache, const t3_kv4_batch* batch, void* k_dev, void* v_dev, int32_t dtype,
                              int32_t layer, int32_t n_layers, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (kv4_check_cache(cache, layer, n_layers, st) || kv4_check_batch(batch)) return 1;
    T3_REQUIRE(k_dev && v_dev, "kv4_read: null argument");
    T3_REQUIRE(dtype == 0 || dtype == 1, "kv4_read: dtype must be 0 (bf16) or 1 (fp16)");
    T3_REQUIRE(reinterpret_cast<uintptr_t>(k_dev) % 16 == 0 && reinterpret_cast<uintptr_t>(v_dev) % 16 == 0, "kv4_read: rows must be 16-byte aligned");
    uint16_t* k = static_cast<uint16_t*>(k_dev);
    uint16_t* v = static_cast<uint16_t*>(v_dev);
    if (cache->hd == 64 && dtype == 0) kv4_read_launch<64, false>(cache, batch, layer, n_layers, k, v, st);
    else if (cache->hd == 64) kv4_read_launch<64, true>(cache, batch, layer, n_layers, k, v, st);
    else if (dtype == 0) kv4_read_launch<128, false>(cache, batch, layer, n_layers, k, v, st);
    else kv4_read_launch<128, true>(cache, batch, layer, n_layers, k, v, st);
    T3_HIP_CHECK(hipGetLastError());
    return 0;
}

template <int HD> static void kv4_evict_launch(const Kv4View& c, const Kv4Evict& e, int layers, int64_t layer_stride, hipStream_t st) {
    const dim3 grid(c.Hkv, e.n, layers);
    // Pages moved by the workgroup that chose them, up to 2048 entries: 4 streams of 2000 x 16 heads of 64 10.5 us, 8 streams x 30 layers
    // 158; moved by a launch of their own 12.3 and 209.  Above, few workgroups would move many pages: one stream of 8000 to 6000 x 8 heads
    // of 128 17 us, moved by those that chose 71.  Above 16384 the weights are not held: 4 streams of 8000 18.5 us held, 36.9 not; of
    // 16000 32 and 67.
    if (e.max_ctx <= 2048) {
        T3_LAUNCH((kv4_evict_kernel<HD, 256, 8, true>), grid, dim3(256), 0, st, c, e, layer_stride);
        return;
    }
    if (e.max_ctx <= 8192) T3_LAUNCH((kv4_evict_kernel<HD, 1024, 8, false>), grid, dim3(1024), 0, st, c, e, layer_stride);
    else if (e.max_ctx <= 16384) T3_LAUNCH((kv4_evict_kernel<HD, 1024, 16, false>), grid, dim3(1024), 0, st, c, e, layer_stride);
    else T3_LAUNCH(kv4_choose_kernel, grid, dim3(KV4_CHOOSE_THREADS), 0, st, c, e);
    const int most = e.keep < e.max_ctx ? e.keep : e.max_ctx;
    T3_LAUNCH(kv4_move_kernel<HD>, dim3((most + 4 * KV4_PAGE - 1) / (4 * KV4_PAGE), c.Hkv * e.n, layers), dim3(256), 0, st, c, e, layer_stride);
}

extern "C" int t3_op_kv4_evict(const t3_kv4_cache* cache, const t3_kv4_evict_desc* d, void* stream) {
    hipStream_t st = static_cast<hipStream_t>(stream);
    T3_REQUIRE(d != nullptr, "kv4_evict: null argument");
    if (kv4_check_cache(cache, d->layer, d->n_layers, st)) return 1;
    T3_REQUIRE(d->src_dev && d->dst_dev && d->ctx_dev && d->weights_dev && d->new_ctx_dev && d->kept_dev, "kv4_evict: null argument");
    T3_REQUIRE(d->n >= 1 && (int64_t)d->n * cache->Hkv <= 65535, "kv4_evict: 1..65535 entries x key heads per call");
    T3_REQUIRE(d->max_ctx >= 1 && d->max_ctx <= d->weights_stride, "kv4_evict: max_ctx must be 1..weights_stride");
    T3_REQUIRE(d->sink >= 0 && d->recent >= 0 && d->keep >= 1 && (int64_t)d->sink + d->recent <= d->keep, "kv4_evict: sink + recent <= keep, keep >= 1");
    T3_REQUIRE(d->keep <= d->weights_stride, "kv4_evict: keep must be at most weights_stride");
    // (entries are read by workgroups that start while others have finished)
    const auto apart = [&](const int32_t* p) { return p >= d->new_ctx_dev + d->n || d->new_ctx_dev >= p + d->n; };
    T3_REQUIRE(apart(d->src_dev) && apart(d->dst_dev) && apart(d->ctx_dev), "kv4_evict: new_ctx must not overlap src, dst or ctx");
    const Kv4View c = kv4_view(cache, d->layer);
    const Kv4Evict e{d->src_dev, d->dst_dev, d->ctx_dev, d->weights_dev, d->weights_stride, d->new_ctx_dev, d->kept_dev,
                     d->n, d->max_ctx, d->keep, d->sink, d->recent};
    if (cache->hd == 64) kv4_evict_launch<64>(c, e, d->n_layers, cache->layer_stride, st);
    else kv4_evict_launch<128>(c, e, d->n_layers, cache->layer_stride, st);
    T3_HIP_CHECK(hipGetLastError());
    return 0;
}
