// 4-bit KV cache: append (quantise and write rows), read (rows back as values), eviction by accumulated attention weight, and
// the checks that every entry point of the cache shares.  Byte order: kv4_layout.h; attention: kv4_attn.hip.
#include "kv4_common.h"

// ------------------------------------------------------------------------------------------------------------------
// Append.  For each row, key head and block of 32 dims, with a = max |x|:
//   2^e = the smallest power of two with a / 2^e < 7,   code = e2m1 value nearest to x / 2^e (ties to the even code).
// A thread takes 8 dims of K and the same of V (two 16-byte loads); the maximum of a block is 4 lanes of butterflies over the
// bits of |x|, which order like the values; the conversion rounds, scales and packs two values at a time.
// ------------------------------------------------------------------------------------------------------------------
template <bool F16> __device__ __forceinline__ void kv4_load8(const void* p, float x[8]) {
    const u32x4 v = *static_cast<const u32x4*>(p);
    if constexpr (F16) {
        const f16x8 h = __builtin_bit_cast(f16x8, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
    } else {
        unpack8(v, x);
    }
}
__device__ __forceinline__ unsigned kv4_absmax_bits(const float x[8]) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) { const unsigned u = __float_as_uint(x[i]) & 0x7fffffffu; m = m > u ? m : u; }
    return m;
}
__device__ __forceinline__ unsigned kv4_lane_max(unsigned v, int off) {
    const unsigned o = (unsigned)__shfl_xor((int)v, off);
    return v > o ? v : o;
}
__device__ __forceinline__ unsigned kv4_codes8(const float x[8], float scale) {
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[0], x[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[2], x[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[4], x[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[6], x[7], scale, 3);
    return r;
}

template <int HD, bool F16>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4View c, Kv4Rows b, const uint16_t* __restrict__ k,
                                                         const uint16_t* __restrict__ v, int64_t k_stride, int64_t v_stride) {
    constexpr int T = HD / 8;                                    // threads of one (row, head)
    const Kv4Seq s = kv4_seq_of(b, c, blockIdx.y);
    if (s.state) return;
    const int n = s.n < b.max_rows ? s.n : b.max_rows;
    const int64_t items = (int64_t)n * c.Hkv * T, step = (int64_t)gridDim.x * 256;
    // all lanes of a wave walk together: the butterflies below read every lane of a (row, head)
    for (int64_t i0 = (int64_t)blockIdx.x * 256; i0 < items; i0 += step) {
        const int64_t i = i0 + threadIdx.x;
        const int ch = (int)(i % T) * 8, h = (int)(i / T % c.Hkv);
        const int64_t j = i / ((int64_t)T * c.Hkv);
        const int64_t slot = (int64_t)s.ctx - s.n + j;
        bool put = i < items && slot >= 0;
        int page = -1;
        if (put) page = c.table[(int64_t)s.stream * c.max_pages + slot / KV4_PAGE];
        put = put && kv4_page_ok(page, c.n_pages);
        float kx[8], vx[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) { kx[e] = 0.f; vx[e] = 0.f; }
        if (put) {
            kv4_load8<F16>(k + (s.start + j) * k_stride + h * HD + ch, kx);
            kv4_load8<F16>(v + (s.start + j) * v_stride + h * HD + ch, vx);
        }
        unsigned ka = kv4_absmax_bits(kx), va = kv4_absmax_bits(vx);
        ka = kv4_lane_max(kv4_lane_max(ka, 1), 2);               // of the block of 32
        va = kv4_lane_max(kv4_lane_max(va, 1), 2);
        unsigned any = ka > va ? ka : va;                        // of the entry
#pragma unroll
        for (int o = 4; o < T; o <<= 1) any = kv4_lane_max(any, o);
        const bool bad = any >= 0x7f800000u;                     // a NaN or an infinity somewhere in the entry
        if (!put) continue;
        const int kb = kv4_scale_byte(ka), vb = kv4_scale_byte(va);
        const unsigned kc = bad ? 0u : kv4_codes8(kx, kv4_scale(kb)), vc = bad ? 0u : kv4_codes8(vx, kv4_scale(vb));
        uint8_t* slab = c.pool + ((int64_t)page * c.Hkv + h) * kv4_slab_bytes(HD);
        const int t = (int)(slot % KV4_PAGE);
        *reinterpret_cast<unsigned*>(slab + kv4_k_at(HD, t, ch)) = kc;
        *reinterpret_cast<uint16_t*>(slab + kv4_v_at(HD, t, ch)) = (uint16_t)vc;
        *reinterpret_cast<uint16_t*>(slab + kv4_v_at(HD, t, ch + 4)) = (uint16_t)(vc >> 16);
        if (ch % KV4_BLOCK == 0) {
            slab[kv4_ks_at(HD, t, ch)] = (uint8_t)(bad ? KV4_NAN_SCALE : kb);
            slab[kv4_vs_at(HD, t, ch)] = (uint8_t)(bad ? KV4_MIN_SCALE : vb);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Read: the inverse, a thread 8 dims of K and of V.
// ------------------------------------------------------------------------------------------------------------------
template <bool F16> __device__ __forceinline__ u32x4 kv4_values8(unsigned codes, unsigned byte, bool nan) {
    const float sc = nan ? __uint_as_float(0x7f800000u) : kv4_scale(byte);
    u32x4 o = {kv4_pair<0>(codes, sc), kv4_pair<1>(codes, sc), kv4_pair<2>(codes, sc), kv4_pair<3>(codes, sc)};
    if constexpr (F16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float lo = bf_lo(o[i]), hi = bf_hi(o[i]);
            // a value appended from fp16 can stand for up to 6 * 2^14: cut at the type's largest instead of becoming infinite
            if (lo == lo) lo = fminf(fmaxf(lo, -65504.f), 65504.f);
            if (hi == hi) hi = fminf(fmaxf(hi, -65504.f), 65504.f);
            const f16x2 p = {(_Float16)lo, (_Float16)hi};
            o[i] = __builtin_bit_cast(unsigned, p);
        }
    }
    return o;
}

template <int HD, bool F16>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4View c, Kv4Rows b, int64_t layer_stride, uint16_t* __restrict__ k,
                                                       uint16_t* __restrict__ v) {
    constexpr int T = HD / 8;
    const Kv4Seq s = kv4_seq_of(b, c, blockIdx.y);
    if (s.state == 1) return;
    const uint8_t* pool = c.pool + (int64_t)blockIdx.z * layer_stride;
    const int n = s.n < b.max_rows ? s.n : b.max_rows;
    const int64_t items = (int64_t)n * c.Hkv * T, step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < items; i += step) {
        const int ch = (int)(i % T) * 8, h = (int)(i / T % c.Hkv);
        const int64_t j = i / ((int64_t)T * c.Hkv), slot = (int64_t)s.ctx - s.n + j;
        const int64_t at = (((int64_t)blockIdx.z * b.rows + s.start + j) * c.Hkv + h) * HD + ch;
        const u32x4 zero = {0u, 0u, 0u, 0u};
        u32x4 ko = zero, vo = zero;
        bool nan = s.state == 2;
        if (!nan && slot >= 0) {
            const int page = c.table[(int64_t)s.stream * c.max_pages + slot / KV4_PAGE];
            nan = !kv4_page_ok(page, c.n_pages);
            const uint8_t* slab = pool + ((int64_t)(nan ? 0 : page) * c.Hkv + h) * kv4_slab_bytes(HD);
            const int t = (int)(slot % KV4_PAGE);
            const unsigned kc = *reinterpret_cast<const unsigned*>(slab + kv4_k_at(HD, t, ch));
            const unsigned vc = *reinterpret_cast<const uint16_t*>(slab + kv4_v_at(HD, t, ch)) |
                                (unsigned)*reinterpret_cast<const uint16_t*>(slab + kv4_v_at(HD, t, ch + 4)) << 16;
            const unsigned kb = slab[kv4_ks_at(HD, t, ch)], vb = slab[kv4_vs_at(HD, t, ch)];
            nan = nan || kb == KV4_NAN_SCALE;
            ko = kv4_values8<F16>(kc, kb, nan);
            vo = kv4_values8<F16>(vc, vb, nan);
        } else if (nan) {
            ko = kv4_values8<F16>(0u, 0u, true);
            vo = ko;
        }
        *reinterpret_cast<u32x4*>(k + at) = ko;
        *reinterpret_cast<u32x4*>(v + at) = vo;
    }
}

// ------------------------------------------------------------------------------------------------------------------
// Eviction, two launches.
//
// Choice: one workgroup per (entry, key head, layer).  Of the c entries, [0, sink) and [c - recent, c) stay; among the others
// the `need` largest weights are found exactly by four rounds of an 8-bit radix histogram over order-preserving keys (ties go to
// the lower index, so the result is a set that any correct sort would give), then the kept indices are written in order.
// Move: one workgroup per (destination page, key head, entry and layer) gathers its 64 tokens' bytes.
// ------------------------------------------------------------------------------------------------------------------
#define KV4_CHOOSE_THREADS 1024

struct Kv4Evict {
    const int32_t* src; const int32_t* dst; const int32_t* ctx;
    float* weights; int64_t weights_stride;
    int32_t* new_ctx; int32_t* kept;
    int n, max_ctx, keep, sink, recent;
};

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

__global__ __launch_bounds__(KV4_CHOOSE_THREADS) void kv4_choose_kernel(Kv4View c, Kv4Evict e) {
    __shared__ int hist[256];
    __shared__ int wave_sums[KV4_CHOOSE_THREADS / 64];
    __shared__ int pick[2];
    const int h = blockIdx.x, i = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x;
    const int src = e.src[i], dst = e.dst[i], ctx = e.ctx[i];
    int32_t* kept = e.kept + (((int64_t)layer * e.n + i) * c.Hkv + h) * e.keep;

    // what refuses the entry; every workgroup of the entry comes to the same answer
    bool bad = src < 0 || src >= c.n_streams || dst < 0 || dst >= c.n_streams || src == dst || ctx < 0 || ctx > e.max_ctx ||
               ctx > (int64_t)c.max_pages * KV4_PAGE;
    const int left = ctx < e.keep ? ctx : e.keep;
    for (int o = tid; o < e.n; o += KV4_CHOOSE_THREADS) bad = bad || (o < i && e.dst[o] == dst) || e.src[o] == dst;
    if (!bad) {
        const int32_t* sp = c.table + (int64_t)src * c.max_pages;
        const int32_t* dp = c.table + (int64_t)dst * c.max_pages;
        const int ns = (ctx + KV4_PAGE - 1) / KV4_PAGE, nd = (left + KV4_PAGE - 1) / KV4_PAGE;
        for (int o = tid; o < ns; o += KV4_CHOOSE_THREADS) {
            const int page = sp[o];
            bad = bad || !kv4_page_ok(page, c.n_pages);
            for (int d = 0; d < nd; ++d) bad = bad || dp[d] == page;
        }
        for (int d = tid; d < nd; d += KV4_CHOOSE_THREADS) bad = bad || !kv4_page_ok(dp[d], c.n_pages);
    }
    if (__syncthreads_or(bad)) {
        for (int j = tid; j < e.keep; j += KV4_CHOOSE_THREADS) kept[j] = -1;
        if (h == 0 && layer == 0 && tid == 0) e.new_ctx[i] = -1;
        return;
    }
    const float* w = e.weights + (((int64_t)layer * c.n_streams + src) * c.Hkv + h) * e.weights_stride;
    float* wd = e.weights + (((int64_t)layer * c.n_streams + dst) * c.Hkv + h) * e.weights_stride;

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
    for (int j = left + tid; j < e.keep; j += KV4_CHOOSE_THREADS) kept[j] = -1;
    for (int64_t j = left + tid; j < e.weights_stride; j += KV4_CHOOSE_THREADS) wd[j] = 0.f;
    if (h == 0 && layer == 0 && tid == 0) e.new_ctx[i] = left;
}

template <int HD>
__global__ __launch_bounds__(256) void kv4_move_kernel(Kv4View c, Kv4Evict e, int64_t layer_stride) {
    __shared__ const uint8_t* from[KV4_PAGE];                    // slab of the old entry that becomes token t, null: none
    __shared__ uint8_t old_t[KV4_PAGE];
    const int h = blockIdx.y % c.Hkv, i = blockIdx.y / c.Hkv, layer = blockIdx.z, tid = threadIdx.x;
    const int left = e.new_ctx[i], j0 = blockIdx.x * KV4_PAGE;
    if (j0 >= left) return;                                      // covers a refused entry (-1)
    uint8_t* pool = c.pool + (int64_t)layer * layer_stride;
    const int32_t* kept = e.kept + (((int64_t)layer * e.n + i) * c.Hkv + h) * e.keep;
    constexpr int slab_bytes = KV4_PAGE * (HD + HD / 16);
    if (tid < KV4_PAGE) {
        const int old = j0 + tid < left ? kept[j0 + tid] : -1;
        from[tid] = old < 0 ? nullptr
                            : pool + ((int64_t)c.table[(int64_t)e.src[i] * c.max_pages + old / KV4_PAGE] * c.Hkv + h) * slab_bytes;
        old_t[tid] = (uint8_t)(old < 0 ? 0 : old % KV4_PAGE);
    }
    __syncthreads();
    uint8_t* to = pool + ((int64_t)c.table[(int64_t)e.dst[i] * c.max_pages + blockIdx.x] * c.Hkv + h) * slab_bytes;
    // K: pieces of one token and lane group, hd / 8 bytes
    typedef typename std::conditional<HD == 64, u32x2, u32x4>::type piece_t;
    {
        const int t = tid & 63, d = (tid >> 6) * (HD / 4);
        const uint8_t* p = from[t];
        piece_t x = {};
        if (p) x = *reinterpret_cast<const piece_t*>(p + kv4_k_at(HD, old_t[t], d));
        *reinterpret_cast<piece_t*>(to + kv4_k_at(HD, t, d)) = x;
    }
    // V: four dims of eight tokens, 16 bytes; two bytes from each
    for (int q = tid; q < 2 * HD; q += 256) {
        const int t0 = q % 8 * 8, d = q / 8 * 4;
        u32x4 x = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint8_t* p = from[t0 + j];
            if (p) x[j / 2] |= (unsigned)*reinterpret_cast<const uint16_t*>(p + kv4_v_at(HD, old_t[t0 + j], d)) << (16 * (j & 1));
        }
        *reinterpret_cast<u32x4*>(to + kv4_v_at(HD, t0, d)) = x;
    }
    // scales: K's blocks, then V's, which follow them
    for (int q = tid; q < 4 * HD; q += 256) {
        const int t = q % KV4_PAGE, d = q / KV4_PAGE * KV4_BLOCK;
        const uint8_t* p = from[t];
        to[kv4_ks_at(HD, t, d)] = p ? p[kv4_ks_at(HD, old_t[t], d)] : (uint8_t)KV4_MIN_SCALE;
    }
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

// workgroups along the rows of a sequence: one per 256 threads' work, capped (the kernels stride over the rest)
static int row_groups(const t3_kv4_cache* c, const t3_kv4_batch* b) {
    const int64_t g = ((int64_t)b->max_rows * c->Hkv * (c->hd / 8) + 255) / 256;
    return (int)(g < 4096 ? g : 4096);
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
    const dim3 grid(row_groups(cache, batch), batch->n_seqs);
    const Kv4View c = kv4_view(cache, layer);
    const Kv4Rows b = kv4_rows(batch);
    const uint16_t* k = static_cast<const uint16_t*>(k_dev);
    const uint16_t* v = static_cast<const uint16_t*>(v_dev);
    if (cache->hd == 64 && dtype == 0) T3_LAUNCH((kv4_append_kernel<64, false>), grid, dim3(256), 0, st, c, b, k, v, k_stride, v_stride);
    else if (cache->hd == 64) T3_LAUNCH((kv4_append_kernel<64, true>), grid, dim3(256), 0, st, c, b, k, v, k_stride, v_stride);
    else if (dtype == 0) T3_LAUNCH((kv4_append_kernel<128, false>), grid, dim3(256), 0, st, c, b, k, v, k_stride, v_stride);
    else T3_LAUNCH((kv4_append_kernel<128, true>), grid, dim3(256), 0, st, c, b, k, v, k_stride, v_stride);
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
    const dim3 grid(row_groups(cache, batch), batch->n_seqs, n_layers);
    const Kv4View c = kv4_view(cache, layer);
    const Kv4Rows b = kv4_rows(batch);
    uint16_t* k = static_cast<uint16_t*>(k_dev);
    uint16_t* v = static_cast<uint16_t*>(v_dev);
    const int64_t ls = cache->layer_stride;
    if (cache->hd == 64 && dtype == 0) T3_LAUNCH((kv4_read_kernel<64, false>), grid, dim3(256), 0, st, c, b, ls, k, v);
    else if (cache->hd == 64) T3_LAUNCH((kv4_read_kernel<64, true>), grid, dim3(256), 0, st, c, b, ls, k, v);
    else if (dtype == 0) T3_LAUNCH((kv4_read_kernel<128, false>), grid, dim3(256), 0, st, c, b, ls, k, v);
    else T3_LAUNCH((kv4_read_kernel<128, true>), grid, dim3(256), 0, st, c, b, ls, k, v);
    T3_HIP_CHECK(hipGetLastError());
    return 0;
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
    const Kv4View c = kv4_view(cache, d->layer);
    const Kv4Evict e{d->src_dev, d->dst_dev, d->ctx_dev, d->weights_dev, d->weights_stride, d->new_ctx_dev, d->kept_dev,
                     d->n, d->max_ctx, d->keep, d->sink, d->recent};
    T3_LAUNCH(kv4_choose_kernel, dim3(cache->Hkv, d->n, d->n_layers), dim3(KV4_CHOOSE_THREADS), 0, st, c, e);
    const int most = d->keep < d->max_ctx ? d->keep : d->max_ctx;
    const dim3 grid((most + KV4_PAGE - 1) / KV4_PAGE, cache->Hkv * d->n, d->n_layers);
    if (cache->hd == 64) T3_LAUNCH(kv4_move_kernel<64>, grid, dim3(256), 0, st, c, e, cache->layer_stride);
    else T3_LAUNCH(kv4_move_kernel<128>, grid, dim3(256), 0, st, c, e, cache->layer_stride);
    T3_HIP_CHECK(hipGetLastError());
    return 0;
}
