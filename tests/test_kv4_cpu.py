"""4-bit KV cache without a GPU: the byte order and the bounds arithmetic of csrc/kv4_layout.h compiled for the host, and the
refusals of the C entry points, which come before any GPU call."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

import _kv4
from chatterbox_vllm_amd import _capi
from chatterbox_vllm_amd.kv4_cache import KV4Cache

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
CSRC = os.path.join(ROOT, "chatterbox_vllm_amd", "csrc")

PROGRAM = r"""
#include "kv4_layout.h"
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#define REQUIRE(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
int main() {
    for (int hd = 64; hd <= 128; hd *= 2) {                      // every code and scale has a place of its own, none outside
        const int bytes = kv4_slab_bytes(hd);
        char* used = (char*)calloc(bytes, 1);
        for (int t = 0; t < 64; ++t)
            for (int d = 0; d < hd; ++d) {
                const int at[2] = {kv4_k_at(hd, t, d), kv4_v_at(hd, t, d)};
                for (int i = 0; i < 2; ++i) {
                    REQUIRE(at[i] >= i * 32 * hd && at[i] < (i + 1) * 32 * hd);
                    REQUIRE(!(used[at[i]] & (1 << d % 2)));
                    used[at[i]] |= 1 << d % 2;
                }
                if (d % 32 == 0) {
                    const int sc[2] = {kv4_ks_at(hd, t, d), kv4_vs_at(hd, t, d)};
                    for (int i = 0; i < 2; ++i) { REQUIRE(sc[i] >= 64 * hd && sc[i] < bytes && !used[sc[i]]); used[sc[i]] = 3; }
                }
                printf("%d %d %d %d %d %d\n", hd, t, d, at[0], at[1], kv4_ks_at(hd, t, d));
            }
        for (int i = 0; i < bytes; ++i) REQUIRE(used[i] == 3);
        // pieces that are moved as one word: 8 K dims in 4 bytes, 4 V dims of 8 tokens in 16
        for (int t = 0; t < 64; ++t)
            for (int d = 0; d < hd; d += 8) {
                REQUIRE(kv4_k_at(hd, t, d) % 4 == 0 && kv4_k_at(hd, t, d + 7) == kv4_k_at(hd, t, d) + 3);
                REQUIRE(kv4_v_at(hd, t / 8 * 8, d) % 16 == 0 && kv4_v_at(hd, t, d) == kv4_v_at(hd, t / 8 * 8, d) + 2 * (t % 8));
                REQUIRE(kv4_v_at(hd, t, d + 3) == kv4_v_at(hd, t, d) + 1);
            }
        for (int t = 0; t < 64; ++t)
            for (int d = 0; d < hd; d += hd / 4) REQUIRE(kv4_k_at(hd, t, d) % (hd / 8) == 0 && kv4_k_at(hd, t, d + hd / 4 - 1) == kv4_k_at(hd, t, d) + hd / 8 - 1);
        free(used);
    }
    const int v[] = {-2147483647 - 1, -5, -1, 0, 1, 2, 3, 4, 5, 6, 7, 64, 2147483647};
    const int n = sizeof(v) / sizeof(v[0]);
    for (int a = 0; a < n; ++a) for (int b = 0; b < n; ++b) for (int s = 0; s < n; ++s) for (int c = 0; c < n; ++c)
        for (int rows = 1; rows < 7; rows += 2) for (int most = 1; most <= rows; ++most) {
            const Kv4Seq q = kv4_seq(v[a], v[b], v[s], v[c], rows, most, 4, 64);
            REQUIRE(q.start >= 0 && q.n >= 0 && q.start + q.n <= rows);
            if (q.state == 0) REQUIRE(q.start == v[a] && q.n == v[b] - v[a] && q.n >= 1 && q.n <= most && v[s] >= 0 && v[s] < 4 && v[c] >= 0 && v[c] <= 64);
            if (v[s] < 0) REQUIRE(q.state == 1);
            if (q.n == 0) REQUIRE(q.state == 1);
            if (v[s] >= 0 && v[a] >= 0 && v[b] > v[a] && v[b] <= rows && v[b] - v[a] <= most && v[s] < 4 && v[c] >= 0 && v[c] <= 64) REQUIRE(q.state == 0);
        }
    for (int a = 0; a < n; ++a) REQUIRE(kv4_page_ok(v[a], 5) == (v[a] >= 0 && v[a] < 5));
    float last = 0.f;
    for (unsigned bits = 0; bits < 0x7f800000u; bits += 977) {   // the smallest power of two that leaves it below 7
        float x; memcpy(&x, &bits, 4);
        const int b = kv4_scale_byte(bits);
        REQUIRE(b >= 2 && b <= 252);
        const double s = __builtin_ldexp(1.0, b - 127);
        if (b < 252) REQUIRE(x / s < 7.0);
        if (b > 2) REQUIRE(x / (s / 2) >= 7.0);
        last = x;
    }
    REQUIRE(last > 3e38f);
    const float w[] = {-__builtin_inff(), -3.f, -1e-40f, 0.f, 1e-40f, 1e-30f, 0.5f, 3.f, __builtin_inff()};
    for (int i = 0; i < 9; ++i) for (int j = 0; j < 9; ++j) {
        unsigned x, y; memcpy(&x, &w[i], 4); memcpy(&y, &w[j], 4);
        REQUIRE((kv4_weight_key(x) < kv4_weight_key(y)) == (w[i] < w[j]));
        REQUIRE(kv4_weight_key(x) > kv4_weight_key(0x7fc00000u) && kv4_weight_key(0xffc00000u) == 0);
    }
    REQUIRE(kv4_weight_key(0x80000000u) == kv4_weight_key(0));
    return 0;
}
"""


def test_layout_and_bounds(tmp_path):
    src, exe = tmp_path / "layout.cpp", tmp_path / "layout"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Xlinker", "--no-undefined", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{CSRC}",
                    str(src), "-o", str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, (run.stdout.splitlines() or [run.stderr])[-1] + run.stderr
    got = torch.tensor([[int(x) for x in line.split()] for line in run.stdout.splitlines()])
    for hd in (64, 128):                                         # the byte order that the tests' own model states
        g = got[got[:, 0] == hd]
        t, d = g[:, 1], g[:, 2]
        assert torch.equal(g[:, 3], _kv4.k_at(hd, t, d)) and torch.equal(g[:, 4], _kv4.v_at(hd, t, d))
        assert torch.equal(g[:, 5], 64 * hd + d // 32 * 64 + t)


def test_model_rounds_to_the_nearest_level():
    """The tests' quantiser against a search over all sixteen codes and every scale."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 32, generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-30, 30, (64, 1), generator=g).double())
    codes, b = _kv4.quantise(x)
    held = _kv4.value(codes, b)
    every = torch.cat([_kv4.LEVELS, -_kv4.LEVELS])[None, None] * torch.exp2(b.double() - 127)[..., None]
    assert torch.equal((held - x).abs(), (every - x[..., None]).abs().amin(-1))
    top = x.abs().amax(-1)
    assert (top / torch.exp2(b[:, 0].double() - 127) < 7).all() and (top / torch.exp2(b[:, 0].double() - 128) >= 7).all()


def test_struct_layouts():
    assert C.sizeof(_capi.T3Kv4Cache) == 3 * 8 + 6 * 4
    assert C.sizeof(_capi.T3Kv4Batch) == 3 * 8 + 4 * 4
    assert C.sizeof(_capi.T3Kv4EvictDesc) == 7 * 8 + 7 * 4 + 4


A = 1 << 20                                                      # an address that is aligned and never followed


def _cache(**kw):
    d = dict(pool_dev=A, block_table_dev=A, layer_stride=8 * 16 * 4352, n_layers=2, n_pages=8, n_streams=4, max_pages=4, Hkv=16, hd=64)
    d.update(kw)
    return _capi.T3Kv4Cache(**d)


def _batch(**kw):
    d = dict(seq_start_dev=A, stream_dev=A, ctx_dev=A, n_seqs=2, rows=6, max_rows=3, max_ctx=256)
    d.update(kw)
    return _capi.T3Kv4Batch(**d)


def _evict(**kw):
    d = dict(src_dev=A, dst_dev=A, ctx_dev=A, weights_dev=A, weights_stride=256, new_ctx_dev=A + 4096, kept_dev=A, n=2, max_ctx=256, keep=32,
             sink=4, recent=8, layer=0, n_layers=2)
    d.update(kw)
    return _capi.T3Kv4EvictDesc(**d)


B = A + 4096                                                     # another


def _refused(lib, rc, words):
    assert rc != 0
    assert re.search(words, lib.t3_last_error().decode()), lib.t3_last_error()


BAD_CACHES = [(dict(pool_dev=None), "null"), (dict(block_table_dev=None), "null"), (dict(hd=96), "head_dim"), (dict(hd=32), "head_dim"),
              (dict(Hkv=0), "heads"), (dict(Hkv=1025), "heads"), (dict(n_pages=0), "empty"), (dict(n_streams=0), "empty"),
              (dict(max_pages=0), "empty"), (dict(pool_dev=A + 8), "aligned"), (dict(layer_stride=8 * 16 * 4352 - 16), "overlap"),
              (dict(layer_stride=8 * 16 * 4352 + 8), "overlap"), (dict(n_layers=0), "layer"), (dict(max_pages=1 << 25), "entries")]
BAD_BATCHES = [(dict(seq_start_dev=None), "null"), (dict(stream_dev=None), "null"), (dict(ctx_dev=None), "null"), (dict(n_seqs=0), "sequences"),
               (dict(n_seqs=70000), "sequences"), (dict(rows=0), "bounds"), (dict(max_rows=7), "bounds"), (dict(max_rows=0), "bounds"),
               (dict(max_ctx=0), "bounds")]


@pytest.mark.parametrize("cache,batch,words", [(c, {}, w) for c, w in BAD_CACHES] + [({}, b, w) for b, w in BAD_BATCHES])
def test_descriptors_are_refused(cache, batch, words):
    lib = _capi.load()
    c, b = C.byref(_cache(**cache)), C.byref(_batch(**batch))
    _refused(lib, lib.t3_op_kv4_append(c, b, A, A, 1024, 1024, 0, 0, None), words)
    _refused(lib, lib.t3_op_kv4_read(c, b, A, A, 0, 0, 1, None), words)
    _refused(lib, lib.t3_op_attn_kv4(c, b, A, 1024, A, 1024, 16, 0, 0.125, None, 0, A, 1 << 30, 0, None), words)
    assert lib.t3_op_attn_kv4_work_bytes(c, b, 16, 0) == -1
    if not batch:
        _refused(lib, lib.t3_op_kv4_evict(c, C.byref(_evict()), None), words)


@pytest.mark.parametrize("kw,words", [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(layer=2), "layer"),
    (dict(layer=-1), "layer"), (dict(k=A + 2), "aligned"), (dict(v=A + 8), "aligned"), (dict(ks=1023), "aligned"), (dict(vs=1028), "aligned"),
    (dict(ks=512), "overlap"), (dict(ks=-1024), "overlap")])
def test_append_refusals(kw, words):
    lib = _capi.load()
    d = dict(k=A, v=A, ks=1024, vs=1024, dtype=0, layer=0)
    d.update(kw)
    _refused(lib, lib.t3_op_kv4_append(C.byref(_cache()), C.byref(_batch()), d["k"], d["v"], d["ks"], d["vs"], d["dtype"], d["layer"], None), words)


@pytest.mark.parametrize("kw,words", [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(dtype=3), "dtype"), (dict(layer=1, n=2), "layer"), (dict(n=0), "layer"),
    (dict(n=-1), "layer"), (dict(layer=2147483647, n=2), "layer"), (dict(k=A + 8), "aligned")])
def test_read_refusals(kw, words):
    lib = _capi.load()
    d = dict(k=A, v=A, dtype=0, layer=0, n=1)
    d.update(kw)
    _refused(lib, lib.t3_op_kv4_read(C.byref(_cache()), C.byref(_batch()), d["k"], d["v"], d["dtype"], d["layer"], d["n"], None), words)


@pytest.mark.parametrize("kw,words", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(dtype=2), "dtype"), (dict(H=24), "query heads"), (dict(H=0), "query heads"),
    (dict(H=8), "query heads"), (dict(H=16 * 65), "query heads"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(qs=1020), "overlap"), (dict(qs=1028), "aligned"), (dict(os=512), "overlap"), (dict(q=A + 4), "aligned"), (dict(out=A + 8), "aligned"),
    (dict(w=A, ws=255), "weights_stride"), (dict(w=A, ws=256, work=None), "work"), (dict(w=A, ws=256, size=6 * 16 * 8 - 1), "work"),
    (dict(w=A, ws=256, work=A + 8), "work"), (dict(layer=2), "layer")])
def test_attention_refusals(kw, words):
    lib = _capi.load()
    d = dict(q=A, qs=1024, out=A, os=1024, H=16, dtype=0, scale=0.125, w=None, ws=0, work=A, size=1 << 30, layer=0)
    d.update(kw)
    _refused(lib, lib.t3_op_attn_kv4(C.byref(_cache()), C.byref(_batch()), d["q"], d["qs"], d["out"], d["os"], d["H"], d["dtype"], d["scale"],
                                     d["w"], d["ws"], d["work"], d["size"], d["layer"], None), words)


@pytest.mark.parametrize("kw,words", [
    (dict(src_dev=None), "null"), (dict(dst_dev=None), "null"), (dict(ctx_dev=None), "null"), (dict(weights_dev=None), "null"),
    (dict(new_ctx_dev=None), "null"), (dict(kept_dev=None), "null"), (dict(n=0), "entries"), (dict(n=5000), "entries"), (dict(max_ctx=257), "max_ctx"),
    (dict(max_ctx=0), "max_ctx"), (dict(new_ctx_dev=A), "overlap"), (dict(new_ctx_dev=A + 4), "overlap"), (dict(ctx_dev=B + 4), "overlap"), (dict(dst_dev=B - 4), "overlap"),
    (dict(keep=0), "keep"), (dict(sink=25), "sink"), (dict(sink=-1), "sink"), (dict(recent=-1), "sink"),
    (dict(sink=2147483647, recent=2147483647), "sink"), (dict(keep=257), "keep"), (dict(layer=1), "layer"), (dict(n_layers=3), "layer"), (dict(n_layers=0), "layer")])
def test_evict_refusals(kw, words):
    lib = _capi.load()
    _refused(lib, lib.t3_op_kv4_evict(C.byref(_cache()), C.byref(_evict(**kw)), None), words)
    _refused(lib, lib.t3_op_kv4_evict(C.byref(_cache()), None, None), "null")


def test_attention_refuses_what_its_grid_cannot_hold():
    lib = _capi.load()
    cache, batch = _cache(max_pages=1 << 21), _batch(max_ctx=(1 << 26) + 1)
    _refused(lib, lib.t3_op_attn_kv4(C.byref(cache), C.byref(batch), A, 1024, A, 1024, 16, 0, 0.125, None, 0, A, 1 << 60, 0, None), r"2\^26")
    assert lib.t3_op_attn_kv4_work_bytes(C.byref(cache), C.byref(batch), 16, 0) == -1
    assert lib.t3_op_attn_kv4_work_bytes(C.byref(cache), C.byref(_batch(max_ctx=1 << 26)), 16, 0) > 0


def test_sizes():
    lib = _capi.load()
    assert lib.t3_op_kv4_page_bytes(16, 64) == 16 * 4352 and lib.t3_op_kv4_page_bytes(1, 128) == 8704
    assert lib.t3_op_kv4_page_bytes(16, 80) == 0 and lib.t3_op_kv4_page_bytes(0, 64) == 0
    c, b = C.byref(_cache()), C.byref(_batch())
    assert lib.t3_op_attn_kv4_work_bytes(c, b, 16, 0) == 0       # one chunk: nothing to join
    assert lib.t3_op_attn_kv4_work_bytes(c, b, 16, 1) >= 6 * 16 * 8
    c = C.byref(_cache(max_pages=1 << 20))
    assert lib.t3_op_attn_kv4_work_bytes(c, C.byref(_batch(max_ctx=40000)), 16, 0) > 0


class HostCache(KV4Cache):
    """A cache whose tensors lie on the host and whose calls are written down instead of made."""

    def __init__(self, kv, hd, streams, max_pages, pages=8):
        self._lib, self.device, self._index, self._scale, self.calls = _capi.load(), torch.device("cpu"), -1, hd ** -0.5, []
        self.num_kv_heads, self.head_dim, self.num_layers, self.num_pages, self.num_streams, self.max_pages = kv, hd, 1, pages, streams, max_pages
        self._c = _cache(n_layers=1, n_pages=pages, n_streams=streams, max_pages=max_pages, Hkv=kv, hd=hd)
        self._ref = C.byref(self._c)

    def _run(self, fn, *args):
        self.calls.append(args)


def i32(x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("weights", [lambda: torch.zeros(5, 1, 128), lambda: torch.zeros(1, 5, 128).transpose(0, 1),
                                     lambda: torch.zeros(5, 128)[:, None], lambda: torch.zeros(5, 128).as_strided((5, 1, 128), (128, 7, 1))])
def test_a_row_of_weights_is_as_long_as_its_entries(weights):
    """Contiguous tensors of one key head, whose stride along it is any number: stream s lies at s * 128."""
    cache, w = HostCache(1, 64, 5, 2), weights()
    assert w.is_contiguous() and w.shape == (5, 1, 128)
    cache.attend(torch.zeros(1, 2, 64, dtype=torch.bfloat16), cache.batch(i32([0, 1]), i32([4]), i32([100]), rows=1), weights=w)
    assert cache.calls[0][9] == w.data_ptr() and cache.calls[0][10] == 128


def test_a_narrow_row_of_weights_is_no_longer_than_it_is():
    cache, w = HostCache(1, 64, 1, 4), torch.zeros(1, 1, 200)[..., :100]
    assert w.is_contiguous() and w.stride(1) == 200
    cache.attend(torch.zeros(1, 2, 64, dtype=torch.bfloat16), cache.batch(i32([0, 1]), i32([0]), i32([100]), rows=1, max_ctx=100), weights=w)
    assert cache.calls[0][10] == 100                             # the library refuses max_ctx past it


def _work_bytes(kv, hd, n_seqs, rows, max_rows, max_ctx, heads, weights):
    lib = _capi.load()
    cache = _cache(n_layers=1, n_pages=1 << 20, n_streams=4096, max_pages=1 << 20, Hkv=kv, hd=hd)
    return lib.t3_op_attn_kv4_work_bytes(C.byref(cache), C.byref(_batch(n_seqs=n_seqs, rows=rows, max_rows=max_rows, max_ctx=max_ctx)), heads, weights)


MIB = 1 << 20


@pytest.mark.parametrize("kv,hd,n_seqs,rows,max_rows,max_ctx,heads", [
    (16, 64, 64, 64, 64, 1 << 15, 16),                            # a decode step, bounds as they are when none is given
    (16, 64, 64, 64, 1, 1 << 15, 16),
    (8, 128, 64, 320, 5, 16000, 64),                              # drafts on shared key heads
    (8, 128, 16, 32000, 2000, 33000, 8),                          # prompts alone
    (16, 128, 16, 32000, 2000, 33000, 16),
    (8, 128, 16, 4110, 4095, 5001, 32),                           # a prompt among decode rows
    (1024, 128, 65535, 1 << 22, 1 << 16, 1 << 26, 1024),          # the largest bounds
    (1, 64, 1, 1, 1, 1 << 26, 1), (1, 64, 1, 1, 1, 1, 64)])
@pytest.mark.parametrize("weights", [0, 1])
def test_the_work_buffer_is_bounded(kv, hd, n_seqs, rows, max_rows, max_ctx, heads, weights):
    """Chunk states of the columns that there are, at most 512 MiB of converted pages, of scores at most 512 MiB and what the columns
    have; beside them per row what the queries have."""
    group, chunks = heads // kv, -(-max_ctx // 1024)
    columns = kv * min(rows * group, n_seqs * min(64, max_rows * group))
    states = columns * chunks * (hd * 4 + 8)
    kept = min(512 * MIB, columns * min(4 * MIB, (max_ctx + 63) * 4)) + kv * (rows * group + 16 * (n_seqs + 1)) * (hd * 2 + 8)
    images = 512 * MIB if max_rows * group >= 768 else 0
    size = _work_bytes(kv, hd, n_seqs, rows, max_rows, max_ctx, heads, weights)
    assert 0 <= size <= states + (kept if weights else 0) + images + 1024


def test_work_buffers_of_loose_bounds():
    tight, loose = (_work_bytes(16, 64, 64, 64, m, 1 << 15, 16, 1) for m in (1, 64))
    assert tight <= loose <= 2 * tight and loose <= 160 * MIB
    assert _work_bytes(16, 64, 64, 64, 64, 1 << 15, 16, 0) <= 16 * MIB
    assert _work_bytes(64, 64, 4, 1 << 25, 1 << 22, 100, 64 * 64, 1) == -1      # more columns than a call may have


@pytest.mark.parametrize("given", [[], ["EXTRA=-DONE", "BUILD=build_x"], ["EXTRA=-DONE", "PRELOAD="]])
def test_no_build_of_the_cache_has_packed_fp32_instructions(given):
    """Their switch is on every compile line of the cache's kernels, whatever else the build is given."""
    lines = subprocess.run(["make", "-n", "-B", "-C", CSRC, *given], capture_output=True, text=True, check=True).stdout.splitlines()
    lines = [x for x in lines if re.search(r" -c kv4(_attn)?\.hip ", x)]
    assert len(lines) == 2 and all("-Xclang -target-feature -Xclang -packed-fp32-ops" in x for x in lines)
    assert all(("-DONE" in x) == (len(given) > 0) for x in lines)


@pytest.mark.parametrize("rows,kv,layout", [
    (5, 1, lambda x: x.as_strided((5, 1, 64), (64, 320, 1))), (1, 2, lambda x: x.as_strided((1, 2, 64), (3, 64, 1))),
    (1, 1, lambda x: x.as_strided((1, 1, 64), (5, 9, 1))), (5, 2, lambda x: x)])
def test_rows_of_any_contiguous_layout_are_taken(rows, kv, layout):
    """The stride along a single row or a single head is any number and plays no part."""
    cache = HostCache(kv, 64, 2, 2)
    x = layout(torch.zeros(rows, kv, 64, dtype=torch.bfloat16))
    batch = cache.batch(i32([0, rows]), i32([0]), i32([rows]), rows=rows)
    cache.append(x, x, batch)
    cache.attend(x, batch)
    cache.attend(x, batch, out=x)
    assert x.is_contiguous()
    assert all(call[i] == kv * 64 for call, at in zip(cache.calls, ((4, 5), (3, 5), (3, 5))) for i in at)
