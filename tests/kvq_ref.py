"""The quantised key-value cache and its attention in 64 bits (torch, any
device), the reference of the kvq tests."""
import math

import torch

PAGE = 16
I8, I4 = 2, 3


def row_bytes(kv, hd):
    return hd if kv == I8 else hd // 2


def block_bytes(kv, hd):
    return 2 * PAGE * row_bytes(kv, hd) + 2 * PAGE * 4 * (1 if kv == I8 else 2)


def quantise(kv, x):
    """codes (int64), scale and zero (f64 holding f32 values) of rows [..., hd] of f64."""
    if kv == I8:
        zero = torch.zeros_like(x[..., :1])
        scale = (x.abs().amax(-1, keepdim=True) / 127).float().double()
        lo, hi = -127, 127
    else:
        zero = x.amin(-1, keepdim=True).float().double() + 0.0  # never -0
        scale = ((x.amax(-1, keepdim=True) - zero) / 15).float().double() + 0.0
        lo, hi = 0, 15
    safe = torch.where(scale > 0, scale, torch.ones_like(scale))
    c = torch.where(scale > 0, torch.round((x - zero) / safe), torch.zeros_like(x)).clamp(lo, hi)
    return c.long(), scale, zero


def rotate(x, cos, sin):
    """x [rows, heads, hd], cos/sin [rows, hd/2], all f64."""
    half = x.shape[-1] // 2
    lo, hi = x[..., :half], x[..., half:]
    c, s = cos[:, None], sin[:, None]
    return torch.cat((lo * c - hi * s, hi * c + lo * s), -1)


class Cache:
    """A pool of blocks and a shuffled page table, with 64-bit reads and writes of single rows."""

    def __init__(self, kv, kv_heads, hd, lens, device, seed=0, spare=2, fill="rows", per_seq=None):
        g = torch.Generator().manual_seed(seed)
        self.kv, self.kv_heads, self.hd, self.device = kv, kv_heads, hd, device
        held = [-(-n // PAGE) for n in lens]
        self.seqs, self.per_seq = len(lens), per_seq or max(max(held, default=0), 1)
        self.pages = sum(held) + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        table = torch.full((self.seqs, self.per_seq), -7, dtype=torch.int32)  # entries no row may reach
        for s, n in enumerate(held):
            for j in range(n):
                table[s, j] = order.pop()
        self.table = table.to(device)
        self.block = block_bytes(kv, hd)
        if fill == "noise":  # every byte anything, scales among them NaN and infinities
            self.pool = torch.randint(0, 256, (self.pages, kv_heads, self.block), dtype=torch.uint8,
                                      generator=g).to(device)
            return
        self.pool = torch.zeros(self.pages, kv_heads, self.block, dtype=torch.uint8, device=device)
        if fill == "rows":
            x = torch.randn(2, self.pages, kv_heads, PAGE, hd, generator=g, dtype=torch.float64)
            x *= torch.exp(0.5 * torch.randn(2, self.pages, kv_heads, PAGE, 1, generator=g, dtype=torch.float64))
            for kind in (0, 1):
                self.put_blocks(kind, x[kind].to(device))

    def codes_view(self, kind):
        rb = row_bytes(self.kv, self.hd)
        return self.pool[..., kind * PAGE * rb:(kind + 1) * PAGE * rb].unflatten(-1, (PAGE, rb))

    def params_view(self, kind):
        n = 1 if self.kv == I8 else 2
        at = 2 * PAGE * row_bytes(self.kv, self.hd) + kind * n * PAGE * 4
        return self.pool[..., at:at + n * PAGE * 4].view(torch.float32).unflatten(-1, (n, PAGE))

    def put_blocks(self, kind, x):
        c, s, z = quantise(self.kv, x)
        self.codes_view(kind).copy_(c.to(torch.int8).view(torch.uint8) if self.kv == I8 else
                                    (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8))
        self.params_view(kind)[..., 0, :] = s[..., 0].float()
        if self.kv == I4:
            self.params_view(kind)[..., 1, :] = z[..., 0].float()

    def rows(self, kind, seq, pos):
        """f64 values [n, kv_heads, hd] of positions `pos` (list or tensor) of one sequence."""
        pos = torch.as_tensor(pos, device=self.device)
        page, slot = self.table[seq, pos // PAGE].long(), pos % PAGE
        b = self.codes_view(kind)[page, :, slot]
        if self.kv == I8:
            c = b.view(torch.int8).double()
        else:
            c = torch.stack((b & 15, b >> 4), -1).flatten(-2).double()
        par = self.params_view(kind)[page, :, :, slot].double()
        x = c * par[..., :1]
        return x if self.kv == I8 else x + par[..., 1:]


def attention(cache, q, seq, length):
    """q [nh, hd] f64 over the first `length` positions: out, lse and the bound of a 32-bit evaluation.

    The bound: a score of `hd` products in 32 bits, with q held to 2^-22 and a
    few further roundings, is off by at most ds = (hd + 16) 2^-23 max_j sum_d
    |q_d||k_jd| / sqrt(hd) plus 2^-21 of its own size for the exponent's
    argument; a zero (I4) enters the score and the output as a product of its
    own, so |k| and |v| there count scale * code and zero apart.  Every weight
    is then off by a factor within exp(+-2 ds), and the sums over `length`
    positions, rounded pairwise over at most length/16 + 64 joins, add that
    many roundings of 2^-23; both scale with max |v|."""
    nh, hd = q.shape
    group = nh // cache.kv_heads
    if length <= 0:
        return q.new_zeros(nh, hd), q.new_full((nh,), -math.inf), q.new_zeros(nh, 1)
    k, v = (cache.rows(kind, seq, torch.arange(length)) for kind in (0, 1))
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("hd,phd->hp", q, k) / math.sqrt(hd)
    lse = torch.logsumexp(s, -1)
    out = torch.einsum("hp,phd->hd", torch.exp(s - lse[:, None]), v)
    wide = 1 if cache.kv == I8 else 3
    ds = (hd + 16) * 2.0**-23 * wide * torch.einsum("hd,phd->hp", q.abs(), k.abs()).amax(-1) / math.sqrt(hd)
    ds = ds + 2.0**-21 * s.abs().amax(-1)
    bound = wide * v.abs().amax((0, 2)) * (4 * ds + (length / 16 + 64) * 2.0**-23)
    return out, lse, bound[:, None]
