"""The 4-bit KV cache on the GPU against the plain 64-bit restatement in _kv4.py: bytes and kept indices are exact, attention is
held to bounds that follow from the roundings (_kv4.out_bound, _kv4.weights_bound)."""
import math

import pytest
import torch

import _kv4
from chatterbox_vllm_amd import _capi
from chatterbox_vllm_amd.kv4_cache import KV4Cache, page_bytes

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def starts(rows):
    s = [0]
    for r in rows:
        s.append(s[-1] + r)
    return s


def device_cache(m):
    return KV4Cache(m.kv, m.hd, pool=m.pool.to(DEV), block_table=m.table.to(DEV))


def check_attend(m, cache, rows, ctx, group, dtype, with_weights, streams=None, layer=0, seed=0, qkv=None, batch=None):
    """One call against the model; returns (q, out, weights)."""
    n = len(rows)
    streams = list(range(n)) if streams is None else streams
    H, R = m.kv * group, sum(rows)
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(R, H, m.hd, generator=g) * 1.5).to(DT[dtype])
    s = starts(rows)
    batch = cache.batch(i32(s), i32(streams), i32(ctx), rows=R, max_rows=max(rows), max_ctx=max(ctx)) if batch is None else batch
    w0 = torch.rand(m.table.shape[0], m.kv, m.table.shape[1] * 64, generator=g)
    w = w0.to(DEV) if with_weights else None
    out = cache.attend(q.to(DEV), batch, layer=layer, weights=w)
    torch.cuda.synchronize()
    scale = m.hd ** -0.5
    want_w, added, slack = w0.double().clone(), torch.zeros_like(w0, dtype=torch.float64), torch.zeros_like(w0, dtype=torch.float64)
    for i in range(n):
        k, v = m.get(m.pool, streams[i], torch.arange(ctx[i]), layer)
        ref, p, size, bound = _kv4.attend(q[s[i]:s[i + 1]].double(), k, v, ctx[i], scale)
        err = (out[s[i]:s[i + 1]].cpu().double() - ref).abs()
        tol = _kv4.out_bound(ref, size, bound, ctx[i], DT[dtype], rows[i] * group)
        assert (err <= tol).all(), f"sequence {i} ({rows[i]} rows, {ctx[i]} entries): {(err / tol).max():.2f} of the bound"
        added[streams[i], :, :ctx[i]] += p
        slack[streams[i], :, :ctx[i]] += _kv4.weights_bound(p, torch.zeros_like(p), bound, ctx[i], rows[i] * group)
    if with_weights:
        err = (w.cpu().double() - (want_w + added)).abs()
        tol = slack + (want_w + added) * 2.0 ** -23
        assert (err <= tol).all(), f"weights: {(err / tol.clamp_min(1e-300)).max():.2f} of the bound"
        assert torch.equal(w.cpu()[added == 0], w0[added == 0])
    return q, out, w


# ---- append, read ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd,kv", [(64, 16), (64, 1), (128, 8), (128, 3)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,ctx", [([1], [1]), ([1, 1, 1], [64, 65, 200]), ([5, 64, 1, 130], [5, 128, 1, 193]), ([9, 3], [4, 130])])
def test_append_and_read_bytes(hd, kv, dtype, rows, ctx):
    m = _kv4.Model(hd, kv, 2, 40, 6, 4, seed=1)
    cache = device_cache(m)
    streams, s, R = [4, 1, 5, 2][:len(rows)], starts(rows), sum(rows)
    g = torch.Generator().manual_seed(2)
    buf = torch.randn(R + 2, 3 * kv, hd, generator=g) * torch.exp2(torch.randint(-20, 12, (R + 2, 3 * kv, 1), generator=g).float())
    buf = buf.to(DT[dtype])
    want, held = m.pool.clone(), []
    for i in range(len(rows)):
        slots = torch.arange(ctx[i] - rows[i], ctx[i])
        ok = slots >= 0                                          # rows before entry 0 are not stored
        rk, rv = buf[s[i]:s[i + 1], kv:2 * kv], buf[s[i]:s[i + 1], 2 * kv:]
        k, v = (torch.zeros(rows[i], kv, hd, dtype=torch.float64) for _ in range(2))
        k[ok], v[ok] = m.put(want, streams[i], slots[ok], rk[ok], rv[ok], layer=1)
        held.append((k, v))
    batch = cache.batch(i32(s), i32(streams), i32(ctx), rows=R, max_rows=max(rows), max_ctx=max(ctx))
    dbuf = buf.to(DEV)[:R]                                       # views of a wider buffer
    cache.append(dbuf[:, kv:2 * kv], dbuf[:, 2 * kv:], batch, layer=1)
    torch.cuda.synchronize()
    assert torch.equal(cache.pool.cpu(), want)
    for out in DT:
        top = torch.finfo(DT[out]).max
        k, v = cache.read(batch, layer=1, dtype=DT[out])
        both = cache.read(batch, layer=0, n_layers=2, dtype=DT[out])
        torch.cuda.synchronize()
        for got, two, ref in ((k, both[0], 0), (v, both[1], 1)):
            ref = torch.cat([h[ref] for h in held]).clamp(-top, top).to(DT[out])
            assert torch.equal(got.cpu(), ref) and torch.equal(two[1].cpu(), ref)


@pytest.mark.parametrize("hd", [64, 128])
def test_append_special_values(hd):
    """Zeros, ties, the largest and smallest magnitudes; an entry with a NaN or an infinity becomes a NaN entry, its neighbours do not."""
    kv, m = 2, _kv4.Model(hd, 2, 1, 4, 1, 2, seed=3)
    cache = device_cache(m)
    tiny, big = 2.0 ** -133, torch.finfo(torch.bfloat16).max
    rows = torch.zeros(12, 2 * kv, hd)
    pattern = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    rows[1] = pattern.repeat(hd // 8)
    rows[2] = -rows[1] * 2.0 ** -100
    rows[3] = rows[1] * 2.0 ** 100
    rows[4, :, 0] = 6.96875                                       # the last bf16 below 7; then 7 itself
    rows[5, :, 0], rows[5, :, 1] = 7.0, 0.6
    rows[6] = tiny
    rows[7], rows[7, 0] = big, -big
    rows[8] = 1.0
    rows[8, 0, hd - 1], rows[8, 3, 5] = math.nan, math.inf        # K head 0; V head 1
    rows[9], rows[9, 1, 0] = 2.0, -math.inf                       # K head 1
    rows[10] = 2.0 ** -126 * pattern.repeat(hd // 8)
    rows[11] = -0.0
    rows = rows.to(torch.bfloat16)
    want = m.pool.clone()
    k, v = m.put(want, 0, torch.arange(12), rows[:, :kv], rows[:, kv:])
    batch = cache.batch(i32([0, 12]), i32([0]), i32([12]), rows=12)
    d = rows.to(DEV)
    cache.append(d[:, :kv], d[:, kv:], batch)
    gk, gv = cache.read(batch)
    torch.cuda.synchronize()
    assert torch.equal(cache.pool.cpu(), want)
    for got, ref in ((gk, k), (gv, v)):
        assert torch.equal(torch.nan_to_num(got.cpu().double(), 77.0), torch.nan_to_num(ref, 77.0))
    nan = torch.isnan(gk.cpu())
    assert nan[8].all() and nan[9, 1].all() and not nan[9, 0].any() and not nan[[0, 1, 2, 3, 4, 5, 6, 7, 10, 11]].any()
    # fp16: what rounds up past its largest value is cut there
    h = torch.full((12, 2 * kv, hd), 65504.0, dtype=torch.float16, device=DEV)
    cache.append(h[:, :kv], h[:, kv:], batch)
    assert (cache.read(batch, dtype=torch.float16)[0] == 65504).all() and (cache.read(batch)[0] == 65536).all()


# ---- attention ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd,kv,group", [(64, 16, 1), (64, 2, 5), (128, 2, 1), (128, 2, 8), (128, 1, 16), (64, 1, 33)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("with_weights", [False, True])
def test_decode(hd, kv, group, dtype, with_weights):
    ctx = [1, 2, 63, 64, 65, 500, 512, 513, 1030]
    m = _kv4.Model(hd, kv, 2, 17 * 9 + 2, 9, 17, seed=4)
    for i, t in enumerate(ctx):
        m.fill(i, t, layer=1)
    check_attend(m, device_cache(m), [1] * 9, ctx, group, dtype, with_weights, layer=1)


@pytest.mark.parametrize("hd,ctx", [(64, [8192, 8193, 20000]), (128, [16390, 8100, 9217])])
def test_decode_long(hd, ctx):
    """Lengths at which the chunks change, and many of them."""
    m = _kv4.Model(hd, 1, 1, 3 * 313, 3, 313, seed=5)
    for i, t in enumerate(ctx):
        m.fill(i, t)
    check_attend(m, device_cache(m), [1] * 3, ctx, 2, "bf16", True)


@pytest.mark.parametrize("hd,kv,group,rows,ctx", [
    (64, 2, 1, [5, 1, 8, 3], [5, 70, 600, 2]),                    # the last: rows before entry 0 see nothing
    (128, 3, 8, [5, 2, 8, 4], [700, 130, 8, 65]),
    (64, 1, 1, [64, 65, 63], [64, 65, 640]),                      # both sides of the form for few columns
    (128, 1, 7, [9, 10, 1], [90, 10, 513]),
    (128, 2, 64, [1, 2], [65, 129])])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_drafts_and_mixed_batches(hd, kv, group, rows, ctx, dtype):
    m = _kv4.Model(hd, kv, 1, 4 * 11 + 1, 4, 11, seed=6)
    for i, t in enumerate(ctx):
        m.fill(i, t)
    check_attend(m, device_cache(m), rows, ctx, group, dtype, True)


@pytest.mark.parametrize("hd,kv,group,rows,ctx", [
    (64, 2, 1, [130, 70, 257], [130, 200, 257]),
    (64, 1, 3, [100, 33], [300, 33]),
    (128, 1, 4, [300, 17, 90], [301, 17, 20]),                    # the last: 70 rows see nothing
    (128, 2, 5, [77], [500])])
@pytest.mark.parametrize("dtype,with_weights", [("bf16", True), ("fp16", False), ("fp16", True)])
def test_prompts(hd, kv, group, rows, ctx, dtype, with_weights):
    m = _kv4.Model(hd, kv, 1, 3 * 8 + 1, 3, 8, seed=7)
    for i, t in enumerate(ctx):
        m.fill(i, t)
    check_attend(m, device_cache(m), rows, ctx, group, dtype, with_weights)


@pytest.mark.parametrize("hd,group,rows,ctx", [(64, 3, [300, 5, 130, 21], [300, 1400, 191, 21]), (128, 8, [130, 90, 1, 100], [333, 90, 2000, 164])])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_prompts_with_pages_converted_beforehand(hd, group, rows, ctx, dtype):
    """Batches of long prompts convert their pages in a launch of their own; a prompt alone, or bounds for which that would take too
    much memory, do not.  All give the same bits."""
    m = _kv4.Model(hd, 2, 1, 4 * 32, 4, 32, seed=31)
    for i, t in enumerate(ctx):
        m.fill(i, t)
    cache = device_cache(m)
    q, out, w = check_attend(m, cache, rows, ctx, group, dtype, True)
    s = starts(rows)
    for i in range(4):
        alone = cache.attend(q[s[i]:s[i + 1]].to(DEV), cache.batch(i32([0, rows[i]]), i32([i]), i32([ctx[i]]), rows=rows[i]))
        assert torch.equal(alone, out[s[i]:s[i + 1]]), i
    wide = torch.full((4, 1 << 15), -1, dtype=torch.int32, device=DEV)
    wide[:, :32] = cache.block_table
    loose = KV4Cache(2, hd, pool=cache.pool, block_table=wide)
    assert torch.equal(loose.attend(q.to(DEV), loose.batch(i32(s), i32([0, 1, 2, 3]), i32(ctx), rows=sum(rows))), out)
    # a page that there is not, inside one prompt and behind another's entries
    cache.block_table[0, 2] = -1
    cache.block_table[1, ctx[1] // 64 + 1:] = 4 * 32
    bad = cache.attend(q.to(DEV), cache.batch(i32(s), i32([0, 1, 2, 3]), i32(ctx), rows=sum(rows), max_rows=max(rows), max_ctx=max(ctx)))
    first = max(0, 128 - (ctx[0] - rows[0]))                       # the first row that sees the page
    assert torch.isnan(bad[first:rows[0]]).all() and torch.equal(bad[:first], out[:first]) and torch.equal(bad[rows[0]:], out[rows[0]:])


@pytest.mark.parametrize("rows", [[1, 1, 1, 1], [4, 1, 2, 3], [90, 1, 200, 7]])
def test_rows_do_not_depend_on_the_batch(rows):
    ctx = [700, 65, 1500, 33]
    m = _kv4.Model(64, 2, 1, 4 * 24, 4, 24, seed=8)
    for i, t in enumerate(ctx):
        m.fill(i, t)
    ctx = [max(a, b) for a, b in zip(ctx, rows)]
    cache = device_cache(m)
    q = torch.randn(sum(rows), 6, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    s = starts(rows)
    full = cache.attend(q, cache.batch(i32(s), i32([0, 1, 2, 3]), i32(ctx), rows=sum(rows)))
    for i in range(4):
        alone = cache.attend(q[s[i]:s[i + 1]], cache.batch(i32([0, rows[i]]), i32([i]), i32([ctx[i]]), rows=rows[i], max_ctx=ctx[i]))
        assert torch.equal(alone, full[s[i]:s[i + 1]])


def test_sharp_and_flat_scores():
    """Scores in the hundreds (one entry takes all) and all equal; NaN entries reach the rows that see them and no others."""
    m = _kv4.Model(64, 1, 1, 9, 1, 9, seed=9)
    k, v = torch.randn(513, 1, 64) * 30, torch.randn(513, 1, 64)
    m.put(m.pool, 0, torch.arange(513), k, v)
    check_attend(m, device_cache(m), [1], [513], 1, "bf16", True)
    m.put(m.pool, 0, torch.arange(513), torch.ones(513, 1, 64), v)
    check_attend(m, device_cache(m), [3], [513], 1, "fp16", True)
    for rows in (5, 200):                                         # both forms; the entry of the row before the last two is NaN
        t = 300
        kk = torch.randn(t, 1, 64)
        kk[t - 3, 0, 7] = math.nan
        m.put(m.pool, 0, torch.arange(t), kk, v[:t])
        cache = device_cache(m)
        q = torch.randn(rows, 1, 64).to(torch.bfloat16)
        out = cache.attend(q.to(DEV), cache.batch(i32([0, rows]), i32([0]), i32([t]), rows=rows)).cpu()
        assert torch.isnan(out[-3:]).all()
        ref, _, size, bound = _kv4.attend(q[:-3].double(), *(x[:t - 3] for x in m.get(m.pool, 0, torch.arange(t))), t - 3, 0.125)
        assert ((out[:-3].double() - ref).abs() <= _kv4.out_bound(ref, size, bound, t, torch.bfloat16, rows)).all()


@pytest.mark.parametrize("hd,rows,ctx", [(64, 1, 2000), (128, 3, 70), (64, 130, 130)])
def test_scores_far_below_zero(hd, rows, ctx):
    """Scores of -1.6e32 and below: the maximum is still found, and equal scores still share the weight."""
    m = _kv4.Model(hd, 1, 1, 40, 1, 32, seed=28)
    k = torch.full((ctx, 1, hd), -2.0 ** 44)
    k[5:9] = -2.0 ** 43                                           # the heaviest four
    v = torch.randn(ctx, 1, hd, generator=torch.Generator().manual_seed(29))
    m.put(m.pool, 0, torch.arange(ctx), k, v)
    _, v = m.get(m.pool, 0, torch.arange(ctx))
    cache = device_cache(m)
    q = torch.full((rows, 1, hd), 2.0 ** 60, dtype=torch.bfloat16, device=DEV)
    out = cache.attend(q, cache.batch(i32([0, rows]), i32([0]), i32([ctx]), rows=rows)).cpu().double()
    for j in range(rows):
        sees = ctx - rows + j + 1
        want = v[5:9].mean(0) if sees >= 9 else v[5:sees].mean(0) if sees > 5 else v[:sees].mean(0)
        assert ((out[j] - want).abs() <= v.abs().max() * 2.0 ** -8 * 1.01).all(), j


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype,low,high", [("fp16", 3.3e4, 6.5e4), ("bf16", 2.0 ** 46, 2.0 ** 47)])
@pytest.mark.parametrize("hd,group,rows,ctx", [(64, 2, [1, 3], [700, 2500]), (128, 1, [1, 1], [130, 1500]), (64, 1, [100, 70], [100, 300]), (128, 8, [120, 1], [200, 70]),
                                               (64, 64, [1, 1], [16500, 300])])
def test_large_scores(hd, group, rows, ctx, dtype, low, high, sign):
    """Scores of one sign that are far from powers of two, from 1e10 on: the largest takes everything, equal ones share it.

    q has at most 11 significant bits and k two, each within a factor of two: products and their sums over hd <= 128 dims take at most
    2 + 11 + 1 + 2 + 7 < 24 bits, so the scores of 32 bits are exact, and two that differ do so by more than 10^4 after the scale.  What
    is left are the last roundings: 1 / n and the sums of n equal terms (2^-22 covers them) and the output's own."""
    n, H = len(rows), group
    m = _kv4.Model(hd, 1, 1, n * 260 + 1, n, 260, seed=38)
    g = torch.Generator().manual_seed(39)
    for i, t in enumerate(ctx):
        k = (low + (high - low) * torch.rand(t, 1, hd, generator=g)).to(DT[dtype]).float() * sign
        k[t // 2:t // 2 + 2] = k[t // 2]                          # neighbours that are equal
        m.put(m.pool, i, torch.arange(t), k, torch.randn(t, 1, hd, generator=g).to(torch.bfloat16))
    q = (low + (high - low) * torch.rand(sum(rows), H, hd, generator=g)).to(DT[dtype])
    cache, s = device_cache(m), starts(rows)
    batch = cache.batch(i32(s), i32(list(range(n))), i32(ctx), rows=sum(rows), max_rows=max(rows), max_ctx=max(ctx))
    w = cache.new_weights()[0]
    plain, out = cache.attend(q.to(DEV), batch), cache.attend(q.to(DEV), batch, weights=w).cpu().double()
    assert torch.equal(plain.cpu().double(), out)
    half = torch.finfo(DT[dtype]).eps / 2
    for i in range(n):
        k, v = m.get(m.pool, i, torch.arange(ctx[i]))
        ref, p, size, _ = _kv4.attend(q[s[i]:s[i + 1]].double(), k, v, ctx[i], hd ** -0.5)
        tol = half * ref.abs() + size * 2.0 ** -22 + torch.finfo(DT[dtype]).smallest_normal
        bad = ~((out[s[i]:s[i + 1]] - ref).abs() <= tol)
        assert not bad.any(), f"sequence {i}: {int(bad.any(-1).sum())} of {bad[..., 0].numel()} columns"
        assert ((w[i, :, :ctx[i]].cpu().double() - p).abs() <= p * 2.0 ** -22).all() and (w[i, :, ctx[i]:] == 0).all()


@pytest.mark.parametrize("hd,group,rows,ctx", [(64, 1, 1, 2500), (128, 4, 2, 700), (64, 1, 130, 400), (128, 8, 120, 1100)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("offset", [0, 5 * 2.0 ** 10, 5 * 2.0 ** 15])
def test_a_common_offset_of_the_scores_cancels(hd, group, rows, ctx, dtype, offset):
    """Scores offset + x with x of a few units, x / 8 and offset whole numbers below 2^24: the same softmax as of x.

    The scores of 32 bits are exact.  A difference of two of them is exact, its product with the scale off by 2^-23 of it at most, of
    at most 64 units: each probability is off by 2^-16 and by what its rounding for the second product leaves (_kv4.out_bound)."""
    m = _kv4.Model(hd, 1, 1, 41, 1, 40, seed=40)
    g = torch.Generator().manual_seed(41)
    k = torch.zeros(ctx, 1, hd)
    k[:, 0, 0] = 2.0 ** 10 if offset else 0.0
    k[:, 0, 32:40] = torch.randint(-2, 3, (ctx, 8), generator=g).float()
    m.put(m.pool, 0, torch.arange(ctx), k, torch.randn(ctx, 1, hd, generator=g).to(torch.bfloat16))
    q = torch.zeros(rows, group, hd)
    q[..., 0] = offset / 2.0 ** 10
    q[..., 32:40] = torch.randint(-3, 4, (rows, group, 8), generator=g).float()
    q = q.to(DT[dtype])
    cache = device_cache(m)
    w = cache.new_weights()[0]
    out = cache.attend(q.to(DEV), cache.batch(i32([0, rows]), i32([0]), i32([ctx]), rows=rows), weights=w).cpu().double()
    kk, v = m.get(m.pool, 0, torch.arange(ctx))
    assert torch.equal(kk, k.double())
    ref, p, size, _ = _kv4.attend(q.double(), kk, v, ctx, hd ** -0.5)
    half = torch.finfo(DT[dtype]).eps / 2
    rounding = 2.0 ** -8 if dtype == "bf16" and rows * group > 64 else 2.0 ** -16
    inner = size * (2.0 ** -15 + rounding + (ctx / 16 + 64) * 2.0 ** -24)
    assert ((out - ref).abs() <= half * (ref.abs() + inner) + inner + torch.finfo(DT[dtype]).smallest_normal).all()
    assert ((w[0, :, :ctx].cpu().double() - p).abs() <= p * (2.0 ** -15 + (ctx + rows * group) / 16 * 2.0 ** -24)).all()


@pytest.mark.parametrize("hd,group,rows,ctx", [(64, 1, 1, 1), (128, 2, 3, 1100), (64, 3, 100, 130), (128, 8, 120, 200)])
def test_the_largest_fp16_values_stay_finite(hd, group, rows, ctx):
    """65504 is held as 65536, which fp16 does not have: fp16 outputs are cut as read cuts them, bf16 ones are exact, NaN entries stay NaN."""
    m = _kv4.Model(hd, 2, 1, 20, 1, 18, seed=43)
    v = torch.full((ctx, 2, hd), 65504.0)
    v[..., 1::2] *= -1
    m.put(m.pool, 0, torch.arange(ctx), torch.zeros(ctx, 2, hd), v)
    cache = device_cache(m)
    batch = cache.batch(i32([0, rows]), i32([0]), i32([ctx]), rows=rows)
    sign = torch.tensor([1.0, -1.0]).repeat(hd // 2).to(DEV)
    q = torch.randn(rows, 2 * group, hd, generator=torch.Generator().manual_seed(44)).to(DEV)
    assert (cache.attend(q.half(), batch) == (65504 * sign).half()).all()
    assert (cache.attend(q.bfloat16(), batch) == (65536 * sign).bfloat16()).all()
    k = torch.zeros(1, 2, hd)
    k[0, 0, 0] = math.nan
    m.put(m.pool, 0, torch.tensor([ctx - rows]), k, v[:1])          # of head 0: seen by every row
    bad = device_cache(m)
    out = bad.attend(q.half(), bad.batch(i32([0, rows]), i32([0]), i32([ctx]), rows=rows))
    assert torch.isnan(out[:, :group]).all() and (out[:, group:] == (65504 * sign).half()).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [[1, 2], [90, 1]])
def test_the_loosest_bounds(hd, rows):
    """A table of 2^26 entries a stream, and no other bound: more chunks than a grid has room for, more workgroups than a launch."""
    m = _kv4.Model(hd, 2, 1, 2 * 24, 2, 24, seed=49)
    ctx = [1500, 300]
    for i, t in enumerate(ctx):
        m.fill(i, t)
    cache = device_cache(m)
    q, out, w = check_attend(m, cache, rows, ctx, 2, "bf16", False)
    wide = torch.full((2, 1 << 20), -1, dtype=torch.int32, device=DEV)
    wide[:, :24] = cache.block_table
    loose = KV4Cache(2, hd, pool=cache.pool, block_table=wide)
    n = 2 if sum(rows) < 9 else 20                                # 20 x 2 heads x 4 tiles x 65536 chunks: past 2^23
    batch = loose.batch(i32(starts(rows) + [sum(rows)] * (n - 2)), i32([0, 1] + [-1] * (n - 2)), i32(ctx + [0] * (n - 2)), rows=sum(rows))
    assert torch.equal(loose.attend(q.to(DEV), batch), out)


def test_what_lies_behind_the_last_entry_does_not_matter():
    """Every byte behind the last entry set, scales to NaN among them."""
    outs = []
    for fill in (0, 255):
        m = _kv4.Model(128, 2, 1, 4, 1, 4, seed=10)
        m.pool.fill_(fill)
        for t in (1, 40, 130):
            m.g.manual_seed(t)
            m.fill(0, t)
            outs.append(check_attend(m, device_cache(m), [1], [t], 2, "bf16", True)[1])
            outs.append(check_attend(m, device_cache(m), [min(t, 70)], [t], 2, "bf16", True)[1])
    assert all(torch.equal(a, b) for a, b in zip(outs[:6], outs[6:]))


def test_skipped_rows_and_strides():
    m = _kv4.Model(64, 2, 1, 30, 5, 5, seed=11)
    for i in range(5):
        m.fill(i, 300)
    cache = device_cache(m)
    rows, R = [3, 100, 1, 0, 2], 106
    s = starts(rows)
    batch = cache.batch(i32(s), i32([0, -1, 2, 3, -7]), i32([40, 300, 280, 10, 9]), rows=R + 4)      # four rows behind the last sequence
    wide = torch.randn(R + 4, 9, 64).to(torch.bfloat16).to(DEV)
    out = torch.full((R + 4, 5, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    got = cache.attend(wide[:, 2:6], batch, out=out[:, 1:])
    assert got.data_ptr() == out[:, 1:].data_ptr()
    touched = [0, 1, 2, 103]
    rest = [i for i in range(R + 4) if i not in touched]
    assert (out[rest] == 7).all() and (out[:, 0] == 7).all()
    tight = cache.attend(wide[:, 2:6].contiguous(), batch)
    assert torch.equal(tight[touched], out[touched, 1:])
    before = cache.pool.clone()
    cache.append(wide[:, :2], wide[:, 2:4], batch)
    changed = (cache.pool != before).view(30, -1).any(1).nonzero().view(-1).tolist()
    assert sorted(changed) == sorted({int(m.table[0, 0]), int(m.table[2, 4])})


def test_one_key_head_and_one_row_in_any_contiguous_layout():
    m = _kv4.Model(64, 1, 1, 10, 2, 5, seed=50)
    for i in range(2):
        m.fill(i, 300)
    cache, plain = device_cache(m), device_cache(m)
    x = torch.randn(7, 1, 64, generator=torch.Generator().manual_seed(51)).to(torch.bfloat16).to(DEV)
    apart = x.as_strided((7, 1, 64), (64, 448, 1))
    for y, rows in ((apart, 7), (x[:1].as_strided((1, 1, 64), (5, 9, 1)), 1)):
        assert y.is_contiguous()
        batch, pbatch = (c.batch(i32([0, rows]), i32([1]), i32([290]), rows=rows) for c in (cache, plain))
        cache.append(y, y, batch)
        plain.append(x[:rows], x[:rows], pbatch)
        assert torch.equal(cache.pool, plain.pool) and torch.equal(cache.attend(y, batch), plain.attend(x[:rows], pbatch))


def test_numbers_that_do_not_fit_give_nan_and_store_nothing():
    """The kernels' own checks: nothing outside the buffers is followed, the rows in question are NaN, the others are right."""
    m = _kv4.Model(64, 2, 1, 30, 6, 5, seed=12)
    for i in range(6):
        m.fill(i, 200)
    m.table[3, 1] = 30                                            # a page that there is not; stream 4 has one at the same place
    m.table[4, 1] = -1
    cache = device_cache(m)
    for rows in (1, 100):
        n, R = 7, 7 * rows
        ctx, streams = [200, 200, 321, 200, 100, 100, 200], [0, 6, 2, 3, 4, 1, 5]
        q = torch.randn(R, 2, 64).to(torch.bfloat16).to(DEV)
        batch = cache.batch(i32(starts([rows] * n)), i32(streams), i32(ctx), rows=R, max_rows=rows, max_ctx=320)
        w = torch.zeros(6, 2, 320, device=DEV)
        out = cache.attend(q, batch, weights=w).view(n, rows, 2, 64).cpu()
        for i in (1, 2, 3, 4):
            assert torch.isnan(out[i, -1]).all()
        assert torch.isnan(out[[1, 2]]).all()
        for i in (0, 5, 6):
            ref, _, size, bound = _kv4.attend(q.cpu().double()[i * rows:(i + 1) * rows], *m.get(m.pool, streams[i], torch.arange(ctx[i])), ctx[i], 0.125)
            assert ((out[i].double() - ref).abs() <= _kv4.out_bound(ref, size, bound, 200, torch.bfloat16, rows)).all()
        assert not torch.isnan(w[[0, 1, 2, 5]]).any() and (w[2] == 0).all()
        k, v = cache.read(batch)
        k, v = k.view(n, rows, 2, 64), v.view(n, rows, 2, 64)
        assert torch.isnan(k[[1, 2]]).all() and torch.isnan(v[[1, 2]]).all()
        if rows == 100:                                           # its rows are entries 100 .. 199, the missing page 64 .. 127
            assert torch.isnan(v[3, :28]).all() and torch.isnan(k[3, :28]).all() and not torch.isnan(v[3, 28:]).any()
        before = cache.pool.clone()
        cache.append(q, q, cache.batch(i32(starts([rows] * n)), i32([6, 9, 2, -1, 7, -2, 8]), i32([200, 5, 321, 0, 1, 2, 3]), rows=R, max_ctx=320))
        assert torch.equal(cache.pool, before)
    # a stream whose second page is missing: rows that end in the first see nothing of it
    q = torch.randn(100, 2, 64).to(torch.bfloat16)
    out = cache.attend(q.to(DEV), cache.batch(i32([0, 100]), i32([4]), i32([100]), rows=100)).cpu()
    assert torch.isnan(out[64:]).all() and not torch.isnan(out[:64]).any()
    # more rows than the bound, rows beyond the tensor, sequences out of order
    q = torch.randn(8, 2, 64).to(torch.bfloat16).to(DEV)
    out = torch.full((8, 2, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    cache.attend(q, cache.batch(i32([0, 4, 5]), i32([0, 1]), i32([9, 9]), rows=8, max_rows=3), out=out)
    assert torch.isnan(out[:3]).all() and (out[3] == 7).all() and not torch.isnan(out[4]).any() and (out[5:] == 7).all()
    out.fill_(7.0)
    cache.attend(q, cache.batch(i32([6, 11]), i32([0]), i32([9]), rows=8, max_rows=8), out=out)
    assert torch.isnan(out[6:]).all() and (out[:6] == 7).all()
    out.fill_(7.0)
    cache.attend(q, cache.batch(i32([5, 2, -3]), i32([0, 1]), i32([9, 9]), rows=8), out=out)
    assert (out == 7).all()


@pytest.mark.parametrize("layout", ["transposed", "view", "narrow"])
def test_weights_of_one_key_head_in_any_contiguous_layout(layout):
    """The stride along a single key head is any number: rows go where the tensor has them, what lies around it stays."""
    m = _kv4.Model(64, 1, 1, 15, 3, 5, seed=36)
    for i, t in enumerate((300, 70, 150)):
        m.fill(i, t)
    cache = device_cache(m)
    q = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(37)).to(torch.bfloat16).to(DEV)
    memory = torch.zeros(4 * 3 * 320, device=DEV)
    w = {"transposed": lambda: memory[:960].view(1, 3, 320).transpose(0, 1), "view": lambda: memory[:960].view(3, 320)[:, None],
         "narrow": lambda: memory[:640].view(1, 1, 640)[..., :320]}[layout]()
    if layout == "narrow":                                       # one stream; a bound past the row is refused
        one = KV4Cache(1, 64, pool=cache.pool, block_table=cache.block_table[:1].contiguous())
        with pytest.raises(_capi.T3Error, match="weights_stride"):
            one.attend(q[:1], one.batch(i32([0, 1]), i32([0]), i32([300]), rows=1, max_ctx=320), weights=memory[:640].view(1, 1, 640)[..., :300])
        batch = one.batch(i32([0, 1]), i32([0]), i32([300]), rows=1)
        cache, q = one, q[:1]
    else:
        batch = cache.batch(i32([0, 1, 2, 3]), i32([0, 1, 2]), i32([300, 70, 150]), rows=3, max_rows=1)
    want = cache.new_weights()[0]
    assert w.is_contiguous() and torch.equal(cache.attend(q, batch, weights=w), cache.attend(q, batch, weights=want))
    assert torch.equal(w, want) and (w[:, 0, 0] > 0).all() and (memory[w.numel():] == 0).all()


def test_weights_of_a_stream_that_occurs_twice():
    """Two sequences of one stream (two drafts, say) are added in their order; equal calls give equal bits."""
    m = _kv4.Model(64, 2, 1, 20, 4, 5, seed=13)
    for i in range(4):
        m.fill(i, 300)
    rows, ctx, streams = [1, 3, 2, 1, 90], [250, 300, 120, 300, 290], [2, 0, 2, 2, 0]
    cache = device_cache(m)
    _, _, w = check_attend(m, cache, rows, ctx, 2, "bf16", True, streams=streams)
    for _ in range(3):
        assert torch.equal(check_attend(m, cache, rows, ctx, 2, "bf16", True, streams=streams)[2], w)


@pytest.mark.parametrize("hd,group", [(64, 1), (64, 5), (128, 8), (128, 21)])
def test_weights_of_few_columns_over_many_chunks(hd, group):
    """Scores kept, contexts of one to three chunks, a stream in two sequences; rows of weights that are not a multiple of four long."""
    m = _kv4.Model(hd, 2, 1, 4 * 40, 4, 40, seed=23)
    rows, ctx, streams = [1, 3, 2, 1, 1], [2500, 1025, 1500, 2490, 3], [2, 0, 2, 3, 1]
    for i, t in ((0, 1025), (1, 3), (2, 2500), (3, 2490)):
        m.fill(i, t)
    cache = device_cache(m)
    q, out, w = check_attend(m, cache, rows, ctx, group, "bf16", True, streams=streams)
    assert torch.equal(check_attend(m, cache, rows, ctx, group, "bf16", True, streams=streams)[2], w)
    batch = cache.batch(i32(starts(rows)), i32(streams), i32(ctx), rows=sum(rows), max_rows=3, max_ctx=2500)
    wide, odd = (torch.zeros(4, 2, width, device=DEV) for width in (2560, 2501))
    for one in (wide, odd):
        assert torch.equal(cache.attend(q.to(DEV), batch, weights=one), out)
    assert torch.equal(wide[..., :2501], odd)


@pytest.mark.parametrize("hd,group,rows,ctx,streams", [(64, 64, [1, 1, 1], [17000, 900, 16500], [0, 1, 0]), (128, 32, [2, 1, 40], [16400, 16400, 700], [1, 1, 0])])
def test_weights_of_more_scores_than_are_kept(hd, group, rows, ctx, streams):
    """Few columns over contexts whose scores are formed again, beside ones whose scores are kept, of one stream too."""
    m = _kv4.Model(hd, 1, 1, 2 * 266, 2, 266, seed=35)
    for i in range(2):
        m.fill(i, max(t for t, x in zip(ctx, streams) if x == i))
    check_attend(m, device_cache(m), rows, ctx, group, "bf16", True, streams=streams)


@pytest.mark.parametrize("hd", [64, 128])
def test_weights_where_scores_find_less_room(hd):
    """Bounds under which the scores' share of the work buffer is cut: 1000 sequences, most of them skipped, over a table of 2^21 entries.
    What is kept of the scores and what is formed again follow the room; outputs are the same bits, weights the same sums."""
    m = _kv4.Model(hd, 4, 1, 3 * 40, 3, 40, seed=42)
    rows, ctx, group = [4, 3, 1], [2500, 1000, 2400], 4
    for i, t in enumerate(ctx):
        m.fill(i, t)
    cache = device_cache(m)
    q, out, w = check_attend(m, cache, rows, ctx, group, "bf16", True)
    wide = torch.full((3, 1 << 15), -1, dtype=torch.int32, device=DEV)
    wide[:, :40] = cache.block_table
    loose = KV4Cache(4, hd, pool=cache.pool, block_table=wide)
    s, n = starts(rows) + [8] * 997, 1000
    batch = loose.batch(i32(s), i32([0, 1, 2] + [-1] * 997), i32(ctx + [0] * 997), rows=8, max_rows=4)
    size = cache._lib.t3_op_attn_kv4_work_bytes(loose._ref, batch._ref, 16, 1)
    assert size < 2 << 30
    many = loose.new_weights()[0]
    assert torch.equal(loose.attend(q.to(DEV), batch, weights=many), out)
    tight = cache.new_weights()[0]
    cache.attend(q.to(DEV), cache.batch(i32(starts(rows)), i32([0, 1, 2]), i32(ctx), rows=8, max_rows=4, max_ctx=2500), weights=tight)
    got = many[..., :2560].cpu()
    assert (many[..., 2560:] == 0).all()
    for i, t in enumerate(ctx):
        k, v = m.get(m.pool, i, torch.arange(t))
        a = sum(rows[:i])
        _, p, _, bound = _kv4.attend(q[a:a + rows[i]].double(), k, v, t, hd ** -0.5)
        for x in (got, tight.cpu()):
            assert ((x[i, :, :t].double() - p).abs() <= _kv4.weights_bound(p, p, bound, t, rows[i] * group)).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_rows_beyond_what_one_launch_has_workgroups_for(hd):
    """270000 rows of one sequence at once give the bytes that they give a thousand at a time, and come back."""
    n, pages = 270000, 4219
    caches = [KV4Cache(1, hd, num_pages=pages, block_table=torch.randperm(pages, generator=torch.Generator().manual_seed(24)).to(torch.int32).to(DEV).view(1, -1)) for _ in range(2)]
    g = torch.Generator(device=DEV).manual_seed(25)
    k, v = (torch.randn(n, 1, hd, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    whole = [c.batch(i32([0, n]), i32([0]), i32([n]), rows=n) for c in caches]
    caches[0].append(k, v, whole[0])
    for i in range(0, n, 999):
        part = min(999, n - i)
        caches[1].append(k[i:i + part], v[i:i + part], caches[1].batch(i32([0, part]), i32([0]), i32([i + part]), rows=part))
    assert torch.equal(caches[0].pool, caches[1].pool)
    got = caches[0].read(whole[0])
    for i in (0, 200000, n - 1000):
        part = caches[1].read(caches[1].batch(i32([0, 1000]), i32([0]), i32([i + 1000]), rows=1000))
        assert all(torch.equal(a[i:i + 1000], b) for a, b in zip(got, part))
        assert ((got[0][i:i + 1000].float() - k[i:i + 1000].float()).abs() <= k[i:i + 1000].float().abs().amax(-1, keepdim=True) / 3.5).all()   # half a step


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [[1, 2], [100, 1], [900, 70]])
def test_empty_streams(hd, rows):
    """Streams without entries: nothing is stored, rows get 0, no weight is added, and the sequence beside them is as it is alone."""
    m = _kv4.Model(hd, 1, 1, 60, 3, 20, seed=33)
    m.fill(2, 1000)
    cache = device_cache(m)
    R = sum(rows) + 80
    x = torch.randn(R, 1, hd, generator=torch.Generator().manual_seed(34)).to(torch.bfloat16).to(DEV)
    batch = cache.batch(i32(starts(rows + [80])), i32([0, 1, 2]), i32([0, 0, 1000]), rows=R, max_rows=max(max(rows), 80))
    pool = cache.pool.clone()
    w, w2 = cache.new_weights()[0], cache.new_weights()[0]
    out = cache.attend(x, batch, weights=w)
    alone = cache.attend(x[-80:], cache.batch(i32([0, 80]), i32([2]), i32([1000]), rows=80), weights=w2)
    assert (out[:-80] == 0).all() and torch.equal(out[-80:], alone) and (w[:2] == 0).all()
    assert torch.equal(w[2] != 0, w2[2] != 0)
    cache.append(x[:-80], x[:-80], cache.batch(i32(starts(rows)), i32([0, 1]), i32([0, 0]), rows=R - 80))
    k, v = cache.read(cache.batch(i32(starts(rows)), i32([0, 1]), i32([0, 0]), rows=R - 80))
    assert torch.equal(cache.pool, pool) and (k == 0).all() and (v == 0).all()


@pytest.mark.parametrize("hd,rows,ctx", [(64, [1, 5, 3], [40, 2000, 3]), (128, [200, 1, 70], [200, 3000, 500])])
def test_out_may_be_q(hd, rows, ctx):
    m = _kv4.Model(hd, 2, 1, 3 * 47, 3, 47, seed=26)
    for i, t in enumerate(ctx):
        m.fill(i, t)
    cache = device_cache(m)
    q = torch.randn(sum(rows), 6, hd, generator=torch.Generator().manual_seed(27)).to(torch.bfloat16).to(DEV)
    batch = cache.batch(i32(starts(rows)), i32([0, 1, 2]), i32(ctx), rows=sum(rows), max_rows=max(rows), max_ctx=max(ctx))
    w, w2 = cache.new_weights()[0], cache.new_weights()[0]
    want = cache.attend(q, batch, weights=w)
    assert cache.attend(q, batch, out=q, weights=w2) is q
    assert torch.equal(q, want) and torch.equal(w, w2)


def test_offsets_past_32_bits():
    """A pool of more than 4 GiB, pages at its end."""
    pages = (1 << 32) // page_bytes(8, 128) + 40
    pool = torch.empty(1, pages, page_bytes(8, 128), dtype=torch.uint8, device=DEV)
    table = torch.arange(pages - 1, pages - 9, -1, dtype=torch.int32, device=DEV).view(2, 4)
    small = KV4Cache(8, 128, num_pages=8, block_table=torch.arange(7, -1, -1, dtype=torch.int32, device=DEV).view(2, 4))
    big = KV4Cache(8, 128, pool=pool, block_table=table)
    g = torch.Generator(device=DEV).manual_seed(0)
    k, v, q = (torch.randn(300, h, 128, generator=g, device=DEV).to(torch.bfloat16) for h in (8, 8, 16))
    got = []
    for c in (small, big):
        b = c.batch(i32([0, 200, 300]), i32([0, 1]), i32([200, 250]), rows=300)
        c.pool[:, -8:].zero_()
        c.append(k, v, b)
        w = c.new_weights()
        w[0, 0] += torch.arange(256, device=DEV)
        got.append([c.attend(q, b, weights=w[0]), *c.read(b), w.clone()])
        c.block_table[1] = c.block_table[1].flip(0)
        got[-1] += [*c.evict(i32([0]), i32([1]), i32([200]), 90, 5, 20, w), *c.read(c.batch(i32([0, 90]), i32([1]), i32([90]), rows=90))]
    assert all(torch.equal(a, b) for a, b in zip(*got))
    del pool, big


# ---- eviction ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd,kv,layers", [(64, 3, 2), (128, 2, 1)])
@pytest.mark.parametrize("keep,sink,recent,ctx", [
    (100, 7, 20, [300, 101, 100, 64, 1, 0]), (64, 0, 0, [65, 640, 127, 64, 63, 2]), (1, 0, 0, [5, 1, 640, 0, 64, 65]),
    (30, 10, 20, [31, 200, 30, 29, 640, 11]), (257, 34, 128, [640, 258, 257, 256, 400, 1])])
def test_evict(hd, kv, layers, keep, sink, recent, ctx):
    n = 6
    m = _kv4.Model(hd, kv, layers, 2 * n * 10 + 1, 2 * n, 10, seed=14)
    for layer in range(layers):
        for i, t in enumerate(ctx):
            m.fill(i, t, layer=layer) if t else None
    g = torch.Generator().manual_seed(15)
    w = torch.rand(layers, 2 * n, kv, 640, generator=g)
    w = torch.where(w < 0.3, torch.zeros(()), (w * 20).floor())   # many ties
    w[:, 0, 0, 30:40], w[:, 1, 1, 40:50] = math.nan, math.inf
    w[:, 0, 1, :], w[:, 1, 0, 5] = 0.0, -1.0
    w[:, 0, 1, ::3] = -0.0
    cache = device_cache(m)
    dw = w.to(DEV)
    dst = [11, 6, 8, 7, 10, 9]
    before = cache.pool.clone()
    new, kept = cache.evict(i32(list(range(n))), i32(dst), i32(ctx), keep, sink, recent, dw)
    torch.cuda.synchronize()
    left = [min(t, keep) for t in ctx]
    assert new.tolist() == left
    pool, after = cache.pool.cpu(), dw.cpu()
    used = m.table[:n].flatten().long()
    assert torch.equal(pool[:, used], before.cpu()[:, used]) and torch.equal(torch.nan_to_num(after[:, :n], 9.5), torch.nan_to_num(w[:, :n], 9.5))
    for layer in range(layers):
        for i in range(n):
            held = m.get(m.pool, i, torch.arange(ctx[i]), layer)
            got = m.get(pool, dst[i], torch.arange(left[i]), layer)
            for h in range(kv):
                stay = _kv4.choose(w[layer, i, h].tolist(), ctx[i], keep, sink, recent)
                assert kept[layer, i, h].tolist() == stay + [-1] * (keep - left[i])
                for a, b in zip(got, held):
                    assert torch.equal(a[:, h], b[stay, h])
                assert torch.equal(torch.nan_to_num(after[layer, dst[i], h, :left[i]], 9.5), torch.nan_to_num(w[layer, i, h][stay], 9.5))
                assert (after[layer, dst[i], h, left[i]:] == 0).all()


def test_evict_long_and_nan_entries():
    """More entries than threads of a workgroup take at once; all weights equal, all different; a NaN entry stays one."""
    m = _kv4.Model(64, 2, 1, 2 * 160, 2, 160, seed=16)
    k = torch.randn(10001, 2, 64)
    k[3, 1, 0] = math.nan
    m.put(m.pool, 0, torch.arange(10001), k, k)
    cache = device_cache(m)
    w = cache.new_weights()
    w[0, 0, 1] = torch.rand(160 * 64, device=DEV)
    host = w.cpu()
    new, kept = cache.evict(i32([0]), i32([1]), i32([10001]), 5000, 4, 1000, w)
    for h in range(2):
        stay = _kv4.choose(host[0, 0, h].tolist(), 10001, 5000, 4, 1000)
        assert kept[0, 0, h].tolist() == stay
        held, got = m.get(m.pool, 0, torch.tensor(stay)), m.get(cache.pool.cpu(), 1, torch.arange(5000))
        assert all(torch.equal(torch.nan_to_num(a[:, h], 9.5), torch.nan_to_num(b[:, h], 9.5)) for a, b in zip(got, held))
    assert torch.isnan(cache.read(cache.batch(i32([0, 5]), i32([1]), i32([5]), rows=5))[0][3, 1]).all()


@pytest.mark.parametrize("pages,ctx", [(32, [2048, 2047, 1025, 64, 513, 1, 0]), (33, [2049, 2048, 300]), (128, [8192, 8191, 4097, 640]), (129, [8193, 130]),
                                       (256, [16384, 9001]), (257, [16385, 700])])
@pytest.mark.parametrize("keep,sink,recent", [(500, 34, 100), (1, 0, 0), (1500, 0, 0), (1024, 1000, 24)])
def test_evict_at_every_length(pages, ctx, keep, sink, recent):
    """The choice for entries up to and past each number that the threads of a workgroup hold: weights that differ everywhere, in one
    bit alone, not at all, in sign and exponent, infinite ones, NaN, and ties that reach over all waves."""
    n, kv = len(ctx), 8
    m = _kv4.Model(64, kv, 1, 2 * n * pages, 2 * n, pages, seed=20)
    m.pool.random_(0, 200, generator=torch.Generator().manual_seed(21))
    g = torch.Generator().manual_seed(22)
    width = pages * 64
    w = torch.rand(1, 2 * n, kv, width, generator=g)
    w[:, :, 1] = (w[:, :, 1] * 3).floor()
    w[:, :, 2] = 0.75
    w[:, :, 3] = torch.where(w[:, :, 3] < 0.5, torch.tensor(1.0), torch.tensor(1.0 + 2.0 ** -23))
    w[:, :, 4] = torch.exp((w[:, :, 4] - 0.5) * 160) * torch.where(torch.rand(2 * n, width, generator=g) < 0.3, -1.0, 1.0)
    w[:, :, 5, ::7], w[:, :, 5, 1::5], w[:, :, 5, 2::11] = math.inf, math.nan, -3e38
    w[:, :, 6] = math.nan
    w[:, :, 7] = torch.arange(width) / 7.0
    cache = device_cache(m)
    dw = w.to(DEV)
    new, kept = cache.evict(i32(list(range(n))), i32([n + i for i in range(n)]), i32(ctx), keep, sink, recent, dw)
    left = [min(t, keep) for t in ctx]
    assert new.tolist() == left
    after = dw.cpu()
    stays = {(i, h): _kv4.choose(w[0, i, h].tolist(), ctx[i], keep, sink, recent) for i in range(n) for h in range(kv)}
    for (i, h), stay in stays.items():
        assert kept[0, i, h].tolist() == stay + [-1] * (keep - left[i])
        assert torch.equal(torch.nan_to_num(after[0, n + i, h], 9.5), torch.nan_to_num(torch.cat([w[0, i, h][stay], torch.zeros(width - left[i])]), 9.5))
    old_k, old_v = cache.read(cache.batch(i32([sum(ctx[:i]) for i in range(n + 1)]), i32(list(range(n))), i32(ctx), rows=sum(ctx)))
    new_k, new_v = cache.read(cache.batch(i32([sum(left[:i]) for i in range(n + 1)]), i32([n + i for i in range(n)]), i32(left), rows=sum(left)))
    for (i, h), stay in stays.items():
        for a, b in ((old_k, new_k), (old_v, new_v)):
            assert torch.equal(a[sum(ctx[:i]):][stay, h], b[sum(left[:i]):sum(left[:i + 1]), h])


def test_evict_refuses_entry_by_entry():
    m = _kv4.Model(64, 2, 1, 40, 12, 3, seed=17)
    for i in range(12):
        m.fill(i, 190)
    m.table[3, 2] = m.table[4, 1]                                 # 3 -> 4: a page of both
    m.table[5, 1] = 40                                            # a page that there is not
    m.table[7, 0] = -3
    cache = device_cache(m)
    w = cache.new_weights()
    w += torch.rand(w.shape, device=DEV)
    pool, w0 = cache.pool.clone(), w.clone()
    #      good  range  range  self   pages  page   page   dst again   dst is a src   too long
    src = [0,    12,    0,     1,     3,     5,     0,     1,          0,             0]
    dst = [11,   10,    -1,    1,     4,     6,     7,     11,         3,             9]
    ctx = [190,  100,   100,   100,   190,   190,   190,   190,        190,           193]
    new, kept = cache.evict(i32(src), i32(dst), i32(ctx), 70, 2, 10, w)
    assert new.tolist() == [70] + [-1] * 9
    assert (kept[:, 1:] == -1).all() and (kept[:, 0] >= 0).all()
    own = m.table[11].long().to(DEV)
    others = [p for p in range(40) if p not in own.tolist()]
    assert torch.equal(cache.pool[:, others], pool[:, others]) and torch.equal(w[:, :11], w0[:, :11])
    # one source may go to several destinations
    new, kept = cache.evict(i32([0, 0]), i32([10, 9]), i32([190, 100]), 70, 2, 10, w)
    assert new.tolist() == [70, 70] and kept.max() < 190


def test_evict_refuses_long_entries_with_bad_pages():
    """The page check of entries past 16384, in a pool of more page ids than it marks at a time."""
    n_pages, width = (1 << 19) + 700, 300
    ids = torch.randperm(n_pages, generator=torch.Generator().manual_seed(45))
    ids = torch.cat([ids[ids >= 1 << 19], ids[ids < 1 << 19]])[:12 * width].to(torch.int32)
    table = ids[torch.randperm(12 * width, generator=torch.Generator().manual_seed(46))].view(12, width)
    ctx, keep, sink, recent = [19200, 17000, 19200, 18000, 16385, 19199], 9000, 10, 500
    nd = -(-keep // 64)
    table[6, nd:] = table[0, :width - nd]                         # behind what is written: does not count
    top = (table[1, :17000 // 64] >= 1 << 19).nonzero()[-1, 0]
    table[7, nd - 1] = table[1, top]                              # 1 -> 7: one page of both, with an id behind the first 2^19
    low = (table[2] < 1 << 19).nonzero()[-1, 0]
    table[8, 0] = table[2, low]                                   # 2 -> 8: the same before
    table[9, nd - 1] = n_pages                                    # 3 -> 9: a page that there is not
    table[4, 256] = -5                                            # 4 -> 10: the source's last page
    assert (table[0] >= 1 << 19).any() and (table[0] < 1 << 19).any()
    cache = KV4Cache(1, 64, num_pages=n_pages, block_table=table.to(DEV))
    for i in (0, 5):
        cache.pool[0, table[i].long().to(DEV)] = torch.randint(0, 200, (width, 4352), dtype=torch.uint8, generator=torch.Generator().manual_seed(i)).to(DEV)
    w = cache.new_weights()
    w[0, :6, 0] = torch.rand(6, width * 64, generator=torch.Generator().manual_seed(47)).to(DEV)
    w0, whole = w.cpu(), cache.pool[0, table[5].long().to(DEV)].clone()
    new, kept = cache.evict(i32(list(range(6))), i32([6, 7, 8, 9, 10, 11]), i32(ctx), keep, sink, recent, w)
    assert new.tolist() == [keep, -1, -1, -1, -1, keep]
    assert (kept[0, 1:5] == -1).all() and torch.equal(w.cpu()[0, 7:11], w0[0, 7:11])
    for i in (0, 5):
        stay = _kv4.choose(w0[0, i, 0].tolist(), ctx[i], keep, sink, recent)
        assert kept[0, i, 0].tolist() == stay
        old = cache.read(cache.batch(i32([0, ctx[i]]), i32([i]), i32([ctx[i]]), rows=ctx[i]))
        got = cache.read(cache.batch(i32([0, keep]), i32([6 + i]), i32([keep]), rows=keep))
        assert all(torch.equal(b, a[stay]) for a, b in zip(old, got))
    assert torch.equal(cache.pool[0, table[5].long().to(DEV)], whole)


def test_evict_four_million_entries():
    ctx, keep, sink, recent = (1 << 22) - 5, 3000001, 100, 4000
    pages = 1 << 16
    cache = KV4Cache(1, 64, num_pages=2 * pages, block_table=torch.arange(2 * pages, dtype=torch.int32, device=DEV).flip(0).view(2, pages))
    g = torch.Generator(device=DEV).manual_seed(48)
    cache.pool[0, :, :4096] = torch.randint(0, 256, (4096,), dtype=torch.uint8, generator=g, device=DEV)
    cache.pool[0, :, 4096:] = 127
    cache.pool[0, pages:, 3] = torch.randint(0, 256, (pages,), dtype=torch.uint8, generator=g, device=DEV)
    w = cache.new_weights()
    w[0, 0, 0] = torch.rand(pages * 64, generator=g, device=DEV)
    order = w[0, 0, 0, sink:ctx - recent].argsort(descending=True, stable=True)[:keep - sink - recent].sort().values + sink
    stay = torch.cat([torch.arange(sink, device=DEV), order, torch.arange(ctx - recent, ctx, device=DEV)])
    old = w[0, 0, 0].clone()
    new, kept = cache.evict(i32([0]), i32([1]), i32([ctx]), keep, sink, recent, w)
    assert new.tolist() == [keep] and torch.equal(kept.view(-1).long(), stay)
    assert torch.equal(w[0, 1, 0, :keep], old[stay]) and (w[0, 1, 0, keep:] == 0).all()
    before, after = cache.read(cache.batch(i32([0, ctx]), i32([0]), i32([ctx]), rows=ctx))[0], cache.read(cache.batch(i32([0, keep]), i32([1]), i32([keep]), rows=keep))[0]
    assert torch.equal(after, before[stay])


# ---- the operators together ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd,kv,group", [(64, 4, 1), (128, 2, 4)])
def test_a_stream_from_prompt_to_eviction_and_on(hd, kv, group):
    """Prompt in, attend with weights, decode some tokens, evict, decode on: every step against the 64-bit model."""
    m = _kv4.Model(hd, kv, 2, 60, 6, 8, seed=18)
    cache = device_cache(m)
    g = torch.Generator().manual_seed(19)
    n, layer = 2, 1
    weights = cache.new_weights()
    model_w = torch.zeros(6, kv, 8 * 64, dtype=torch.float64)
    slack = 0.0

    def step(rows, ctx, streams):
        nonlocal slack
        s, R = starts(rows), sum(rows)
        qkv = torch.randn(R, kv * group + 2 * kv, hd, generator=g).to(torch.bfloat16)
        d = qkv.to(DEV)
        q, k, v = d[:, :kv * group], d[:, kv * group:-kv], d[:, -kv:]
        batch = cache.batch(i32(s), i32(streams), i32(ctx), rows=R)
        cache.append(k, v, batch, layer=layer)
        out = cache.attend(q, batch, layer=layer, weights=weights[layer]).cpu().double()
        for i, st in enumerate(streams):
            m.put(m.pool, st, torch.arange(ctx[i] - rows[i], ctx[i]), qkv[s[i]:s[i + 1], kv * group:-kv], qkv[s[i]:s[i + 1], -kv:], layer)
            kk, vv = m.get(m.pool, st, torch.arange(ctx[i]), layer)
            ref, p, size, bound = _kv4.attend(qkv[s[i]:s[i + 1], :kv * group].double(), kk, vv, ctx[i], hd ** -0.5)
            assert ((out[s[i]:s[i + 1]] - ref).abs() <= _kv4.out_bound(ref, size, bound, ctx[i], torch.bfloat16, rows[i] * group)).all()
            model_w[st, :, :ctx[i]] += p
            slack = max(slack, _kv4.weights_bound(p, p, bound, ctx[i], rows[i] * group).max().item())

    ctx = [150, 97]
    step(ctx, ctx, [0, 1])
    steps = 1
    for _ in range(5):
        ctx = [t + 1 for t in ctx]
        step([1, 1], ctx, [0, 1])
        steps += 1
    w = weights[layer].cpu().double()
    assert ((w - model_w).abs() <= 8 * steps * slack).all()
    new, kept = cache.evict(i32([0, 1]), i32([2, 3]), i32(ctx), keep=80, sink=8, recent=16, weights=weights[layer:], layer=layer)
    assert new.tolist() == [80, 80]
    host = weights[layer].cpu()
    for i in range(n):
        for h in range(kv):
            stay = _kv4.choose(w[i, h].tolist(), ctx[i], 80, 8, 16)
            assert kept[0, i, h].tolist() == stay
            assert torch.equal(host[2 + i, h, :80].double(), w[i, h][stay]) and (host[2 + i, h, 80:] == 0).all()
    m.pool = cache.pool.cpu().clone()
    model_w = host.double().clone()
    ctx = [80, 80]
    for _ in range(3):
        ctx = [t + 1 for t in ctx]
        step([1, 1], ctx, [2, 3])
    step([2, 90], [85, 173], [2, 3])
    assert ((weights[layer].cpu().double() - model_w).abs() <= 8 * 5 * slack + model_w * 2.0 ** -21).all()


def test_captured_steps_replay():
    """A decode step (append, attend with weights, read) and an eviction captured into graphs: replays follow what is written into
    the batch's tensors, two graphs do not disturb each other, eager work runs in between."""
    n = 4
    m = _kv4.Model(64, 4, 1, 90, 8, 11, seed=20)
    for i in range(n):
        m.fill(i, 600)
    cache, eager = device_cache(m), device_cache(m)
    g = torch.Generator(device=DEV).manual_seed(21)

    def inputs():
        return torch.randn(n, 16, 64, generator=g, device=DEV).to(torch.bfloat16)

    def step(c, x, b, w):
        c.append(x[:, 8:12], x[:, 12:], b)
        return (c.attend(x[:, :8], b, weights=w), *c.read(b))

    x, ctx, w, we = inputs(), i32([600, 64, 65, 512]), cache.new_weights(), eager.new_weights()
    s, streams = i32(starts([1] * n)), i32(list(range(n)))
    batch, ebatch = cache.batch(s, streams, ctx, rows=n, max_rows=1), eager.batch(s, streams, ctx, rows=n, max_rows=1)
    src, dst, ectx = i32([0, 2]), i32([4, 5]), i32([600, 70])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                                 # warm-up, on scratch weights
        step(cache, x, batch, cache.new_weights()[0])
    torch.cuda.current_stream().wait_stream(side)
    cache.pool.copy_(eager.pool)
    torch.cuda.synchronize()
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        got = step(cache, x, batch, w[0])
    with torch.cuda.graph(two):
        new, kept = cache.evict(src, dst, ectx, 50, 4, 8, w)
    cache.pool.copy_(eager.pool)
    w.zero_()
    for t in range(4):
        x.copy_(inputs())
        ctx.add_(1)
        ectx.copy_(i32([int(ctx[0]), int(ctx[2])]))
        one.replay()
        two.replay()
        torch.cuda.synchronize()
        want = step(eager, x, ebatch, we[0])
        enew, ekept = eager.evict(src, dst, ectx, 50, 4, 8, we)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), t
        assert torch.equal(new, enew) and torch.equal(kept, ekept) and torch.equal(w, we) and torch.equal(cache.pool, eager.pool)


def test_two_streams_at_once():
    """Calls in flight on two streams use work buffers of their own."""
    m = _kv4.Model(64, 4, 1, 4 * 40, 4, 40, seed=22)
    for i in range(4):
        m.fill(i, 2500)
    cache = device_cache(m)
    q = torch.randn(2, 2, 8, 64).to(torch.bfloat16).to(DEV)
    batches = [cache.batch(i32([0, 1, 2]), i32(s), i32([2500, 2400]), rows=2, max_rows=1) for s in ([0, 1], [2, 3])]
    want = [cache.attend(q[i], batches[i]) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(cache.attend(q[i], batches[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_python_refusals():
    cache = KV4Cache(2, 64, num_pages=4, num_streams=2, max_pages=2)
    b = cache.batch(i32([0, 3]), i32([0]), i32([3]), rows=3)
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=DEV)
    w = cache.new_weights()
    other = KV4Cache(2, 64, num_pages=4, num_streams=2, max_pages=2)
    for i, bad in enumerate((lambda: KV4Cache(2, 80, num_pages=1, num_streams=1, max_pages=1), lambda: KV4Cache(2, 64, num_streams=1, max_pages=1),
                lambda: KV4Cache(2, 64, num_pages=1), lambda: KV4Cache(2, 64, pool=cache.pool[:, :, :-1], block_table=cache.block_table),
                lambda: KV4Cache(2, 64, pool=cache.pool[:, ::2], block_table=cache.block_table), lambda: KV4Cache(2, 64, pool=cache.pool.cpu(), block_table=cache.block_table),
                lambda: KV4Cache(2, 64, pool=cache.pool, block_table=cache.block_table.long()), lambda: KV4Cache(2, 64, pool=cache.pool, block_table=cache.block_table.t()),
                lambda: cache.batch(i32([0, 3]), i32([0, 1]), i32([3]), rows=3), lambda: cache.batch(torch.tensor([0, 3], device=DEV), i32([0]), i32([3]), rows=3),
                lambda: cache.batch(i32([0, 3]).cpu(), i32([0]), i32([3]), rows=3),
                lambda: cache.append(x.float(), x, b), lambda: cache.append(x, x.half(), b), lambda: cache.append(x[:2], x[:2], b), lambda: cache.append(x.cpu(), x, b),
                lambda: cache.append(x.transpose(0, 1).contiguous().transpose(0, 1), x, b), lambda: cache.append(x[..., :32], x, b), lambda: cache.append(x, x, other.batch(i32([0, 3]), i32([0]), i32([3]), rows=3)),
                lambda: cache.attend(x[:, :1], b), lambda: cache.attend(x[0], b), lambda: cache.attend(x, b, out=x.half()), lambda: cache.attend(x, b, out=x[:2]),
                lambda: cache.attend(x, b, weights=w), lambda: cache.attend(x, b, weights=w[0].double()), lambda: cache.attend(x, b, weights=w[0, :1]),
                lambda: cache.read(b, dtype=torch.float32), lambda: cache.read(b, n_layers=0),
                lambda: cache.evict(i32([0]), i32([1, 0]), i32([3]), 2, 0, 0, w), lambda: cache.evict(i32([0]), i32([1]), i32([3]), 2, 0, 0, w[0]),
                lambda: cache.evict(i32([0]), i32([1]), i32([3]), 0, 0, 0, w), lambda: cache.evict(i32([0]).long(), i32([1]), i32([3]), 2, 0, 0, w))):
        try:
            bad()
        except ValueError:
            continue
        pytest.fail(f"call {i} was not refused")
    for i, bad in enumerate((lambda: cache.append(x, x, b, layer=1), lambda: cache.attend(x, b, scale=-1.0), lambda: cache.attend(x, b, layer=-1), lambda: cache.read(b, n_layers=2),
                lambda: cache.evict(i32([0]), i32([1]), i32([3]), 2, 2, 1, w), lambda: cache.evict(i32([0]), i32([1]), i32([3]), 500, 2, 1, w),
                lambda: cache.append(torch.zeros(3 * 130, dtype=torch.bfloat16, device=DEV).as_strided((3, 2, 64), (130, 64, 1)), x, b))):
        try:
            bad()
        except _capi.T3Error:
            continue
        pytest.fail(f"call {i} was not refused by the library")
    with pytest.raises(ValueError):
        page_bytes(2, 96)
    torch.cuda.synchronize()
