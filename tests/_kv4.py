"""The 4-bit KV cache restated in plain 64-bit torch on the CPU: format, byte order, attention, choice of what stays."""
import math

import torch

PAGE = 64
LEVELS = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def k_at(hd, t, d):
    two, q = 128 // hd, hd // 4
    return (t % 4 // two) * 1024 + ((d // q) * 16 + t // 4) * 16 + (t % 4 % two) * 8 + d % q // 2


def v_at(hd, t, d):
    return 32 * hd + (d // 64 * 2 + t // 8 % 2) * 1024 + ((t // 16) * 16 + d % 64 // 4) * 16 + t % 8 * 2 + d % 4 // 2


def slab_bytes(hd):
    return PAGE * (hd + hd // 16)


def quantise(x):
    """x [..., hd] -> (codes [..., hd], scale bytes [..., hd / 32]) as int64, by comparison with the midpoints of the levels."""
    x = x.double()
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -125)
    for k in range(-125, 126):                                   # the smallest power of two with top / 2^k < 7
        e = torch.where((top / 2.0 ** k >= 7) & (e <= k), torch.full_like(e, k + 1), e)
    e = e.clamp(-125, 125)
    y = b / torch.exp2(e)
    mid = (LEVELS[1:] + LEVELS[:-1]) / 2
    code = torch.zeros(y.shape, dtype=torch.long)
    for i in range(7):                                           # a tie goes to the even code
        code += (y.abs() >= mid[i]) if i % 2 else (y.abs() > mid[i])
    return (code + 8 * torch.signbit(y)).reshape(x.shape), (e.squeeze(-1) + 127).long()


def value(codes, scales):
    v = LEVELS[codes % 8] * torch.where(codes >= 8, -1.0, 1.0).double()
    return (v.reshape(*v.shape[:-1], v.shape[-1] // 32, 32) * torch.exp2(scales.double() - 127)[..., None]).reshape(v.shape)


class Model:
    """A cache held as values: streams[s][layer] = (K [t, kv, hd], V) in fp64, and its pool as bytes."""

    def __init__(self, hd, kv, layers, pages, streams, max_pages, seed):
        g = torch.Generator().manual_seed(seed)
        self.hd, self.kv, self.layers, self.g = hd, kv, layers, g
        self.pool = torch.randint(0, 256, (layers, pages, kv * slab_bytes(hd)), generator=g, dtype=torch.uint8)
        self.table = torch.randperm(pages, generator=g)[: streams * max_pages].to(torch.int32).view(streams, max_pages)

    def address(self, stream, slots):
        """Offsets [len(slots), kv, hd] of K and V codes and [len(slots), kv, hd / 32] of their scales, in one layer's bytes."""
        hd, t = self.hd, (slots % PAGE)[:, None, None]
        base = (self.table[stream].long()[slots // PAGE][:, None] * self.kv + torch.arange(self.kv))[..., None] * slab_bytes(hd)
        d, nb = torch.arange(hd), torch.arange(hd // 32)
        return base + k_at(hd, t, d), base + v_at(hd, t, d), base + 64 * hd + nb * PAGE + t, base + 66 * hd + nb * PAGE + t

    def put(self, pool, stream, slots, k, v, layer=0):
        """What append does to the bytes; returns the values that are then held."""
        flat = pool[layer].view(-1)
        ka, va, ks, vs = self.address(stream, slots)
        (kc, kb), (vc, vb) = quantise(torch.nan_to_num(k.double(), 0, 0, 0)), quantise(torch.nan_to_num(v.double(), 0, 0, 0))
        bad = ~(torch.isfinite(k.double()).all(-1) & torch.isfinite(v.double()).all(-1))
        kc, vc = (torch.where(bad[..., None], 0, x) for x in (kc, vc))
        kb, vb = torch.where(bad[..., None], 255, kb), torch.where(bad[..., None], 2, vb)
        flat[ka[..., ::2]] = (kc[..., ::2] | kc[..., 1::2] << 4).to(torch.uint8)
        flat[va[..., ::2]] = (vc[..., ::2] | vc[..., 1::2] << 4).to(torch.uint8)
        flat[ks], flat[vs] = kb.to(torch.uint8), vb.to(torch.uint8)
        return self.get(pool, stream, slots, layer)

    def get(self, pool, stream, slots, layer=0):
        flat = pool[layer].view(-1)
        ka, va, ks, vs = self.address(stream, slots)
        odd = torch.arange(self.hd) % 2
        kc, vc = (flat[a].long() >> (4 * odd) & 15 for a in (ka, va))
        kb, vb = flat[ks].long(), flat[vs].long()
        nan = (kb[..., :1] == 255)
        return tuple(torch.where(nan, math.nan, value(c, b)) for c, b in ((kc, kb), (vc, vb)))

    def fill(self, stream, n, layer=0, spread=1.0):
        """Fills entries 0 .. n - 1 of a stream with random rows."""
        k = torch.randn(n, self.kv, self.hd, generator=self.g) * spread
        k[:, :, ::16] *= 4
        v = torch.randn(n, self.kv, self.hd, generator=self.g)
        self.put(self.pool, stream, torch.arange(n), k.to(torch.bfloat16), v.to(torch.bfloat16), layer)


def attend(q, k, v, ctx, scale):
    """q [n, H, hd] (the last rows of ctx entries), k, v [ctx, kv, hd], all fp64 -> out [n, H, hd], weights [kv, ctx], and what the
    tolerances need: sum_t p |v| like out, and the largest error of a score's fp32 sum in units of 2^-24."""
    n, H, hd = q.shape
    kv = k.shape[1]
    out, weights, size = torch.zeros(n, H, hd, dtype=torch.float64), torch.zeros(kv, ctx, dtype=torch.float64), torch.zeros(n, H, hd, dtype=torch.float64)
    bound = 0.0
    for j in range(n):
        sees = ctx - n + j + 1
        if sees <= 0:
            continue
        for h in range(H):
            kk, vv = k[:sees, h * kv // H], v[:sees, h * kv // H]
            s = kk @ q[j, h] * scale
            p = torch.softmax(s, 0)
            out[j, h], size[j, h] = p @ vv, p @ vv.abs()
            weights[h * kv // H, :sees] += p
            if torch.isfinite(s).all():
                bound = max(bound, ((hd + 4) * (kk.abs() @ q[j, h].abs()).max() * scale + 4 * s.abs().max()).item())
    return out, weights, size, bound


def out_bound(ref, size, bound, ctx, dtype, columns=1):
    """|out - ref| may be: half a step of the output; each probability off by twice a score's error (its own and the sum's), by what
    its rounding leaves (half a step of bf16 is 2^-8: one part, as bf16 sequences of more than 64 columns have it; 2^-16 in two), and
    by the fp32 sums over ctx entries."""
    eps = torch.finfo(dtype).eps / 2
    rounding = 2.0 ** -8 if dtype == torch.bfloat16 and columns > 64 else 2.0 ** -16
    inner = size * (2 * bound * 2.0 ** -24 + rounding + (ctx / 16 + 64) * 2.0 ** -24)
    return eps * (ref.abs() + inner) + inner + torch.finfo(dtype).smallest_normal * 2 ** -7


def weights_bound(added, total, bound, ctx, columns):
    """The same for the summed probabilities, added to what was there."""
    return added * (2 * bound + ctx / 16 + columns / 16 + 64) * 2.0 ** -24 + total.abs() * 2.0 ** -24


def choose(w, ctx, keep, sink, recent):
    """Old indices that stay, ascending."""
    if ctx <= keep:
        return list(range(ctx))
    order = sorted(range(sink, ctx - recent), key=lambda t: (-w[t] if w[t] == w[t] else math.inf, t))
    return list(range(sink)) + sorted(order[: keep - sink - recent]) + list(range(ctx - recent, ctx))
