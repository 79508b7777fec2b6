"""The quantised paged key-value cache on the GPU (PagedKV and the quantised
types of a model's KVCache) against 64-bit references: codes and parameters
exactly, attention within the bound of a 32-bit evaluation (kvq_ref)."""
import math

import numpy as np
import pytest

import kvq_ref as R
from bitnetrs_b200 import KV_I4, KV_I8, BackendError, BitNetModel, InvalidConfig, ModelConfig, PagedKV, \
    QuantizationError, synth

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
KINDS = [KV_I8, KV_I4]


class Bench:
    """Device tensors of one cache and the calls on it."""

    def __init__(self, be, cache):
        self.be, self.c, self.dev = be, cache, cache.device
        self.status = torch.zeros(1, dtype=torch.int32, device=self.dev)
        self.kv = PagedKV(be, cache.pool.data_ptr(), cache.table.data_ptr(), pages=cache.pages, seqs=cache.seqs,
                          pages_per_seq=cache.per_seq, kv_heads=cache.kv_heads, head_dim=cache.hd, kv_dtype=cache.kv)

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def space(self, nh):
        return torch.empty(self.kv.attention_workspace(nh), dtype=torch.uint8, device=self.dev).random_(0, 256)

    def store(self, k, v, seq, pos, rope=None, stream=1):
        sq, ps = self.ints(seq), self.ints(pos)
        self.kv.store(k.data_ptr(), v.data_ptr(), k.shape[0], sq.data_ptr(), ps.data_ptr(),
                      self.status.data_ptr(), ldk=k.stride(0), ldv=v.stride(0), bf16=k.dtype == torch.bfloat16,
                      rope=rope, stream=stream)

    def load(self, k, v, seq, pos):
        sq, ps = self.ints(seq), self.ints(pos)
        self.kv.load(k.data_ptr(), v.data_ptr(), k.shape[0], sq.data_ptr(), ps.data_ptr(),
                     self.status.data_ptr(), ldk=k.stride(0), ldv=v.stride(0), bf16=k.dtype == torch.bfloat16, stream=1)

    def attend(self, q, nh, seq, lens, max_len=None, out=None, lse=True):
        out = torch.full_like(q, 77.0) if out is None else out
        ls = torch.full((q.shape[0], nh), 77.0, device=self.dev) if lse else None
        sp = self.space(nh)
        sq, ln = self.ints(seq), self.ints(lens)
        self.kv.attention(q.data_ptr(), out.data_ptr(), q.shape[0], nh, sq.data_ptr(), ln.data_ptr(),
                          max(list(lens) + [0]) if max_len is None else max_len, sp.data_ptr(), sp.numel(),
                          self.status.data_ptr(), ldq=q.stride(0), ldo=out.stride(0), bf16=q.dtype == torch.bfloat16,
                          lse=ls.data_ptr() if lse else 0, stream=1)
        torch.cuda.synchronize()
        return out, ls

    def prompt(self, q, nh, seqs, cu, starts, max_len=None):
        out = torch.full_like(q, 77.0)
        ls = torch.full((q.shape[0], nh), 77.0, device=self.dev)
        sp = self.space(nh)
        a, b, c = self.ints(seqs), self.ints(cu), self.ints(starts)
        most = max([s + cu[i + 1] - cu[i] for i, s in enumerate(starts)])
        self.kv.prompt_attention(q.data_ptr(), out.data_ptr(), q.shape[0], nh, len(seqs), a.data_ptr(), b.data_ptr(),
                                 c.data_ptr(), most if max_len is None else max_len, sp.data_ptr(), sp.numel(),
                                 self.status.data_ptr(), ldq=q.stride(0), ldo=out.stride(0),
                                 bf16=q.dtype == torch.bfloat16, lse=ls.data_ptr(), stream=1)
        torch.cuda.synchronize()
        return out, ls


def bench(be, kv, heads, hd, lens, **kw):
    return Bench(be, R.Cache(kv, heads, hd, lens, torch.device("cuda", be.device_id), **kw))


def check_row(b, q_row, nh, seq, length, out_row, lse_row, fp16_weights=False):
    """fp16_weights: each softmax weight w_j is rounded once to fp16, by at most half a step, 2^-11 w_j, where it
    multiplies the codes' part of v_j: c * scale (I8), or (c - 7.5) * scale (I4), at most half the row's range.  Both are
    at most max |v|, and the weights add up to 1, so the output is off by at most 2^-11 max |v| more."""
    hd = b.c.hd
    ref, lse, bound = R.attention(b.c, q_row.double().view(nh, hd), seq, length)
    if fp16_weights and length > 0:
        bound = bound + 2.0**-11 * b.c.rows(1, seq, range(length)).abs().max()
    got = out_row.double().view(nh, hd)
    if out_row.dtype == torch.bfloat16:
        bound = bound * (1 + 2.0**-8) + 2.0**-8 * ref.abs()
    assert torch.isfinite(got).all()
    over = (got - ref).abs() - bound
    assert (over <= 0).all(), f"seq {seq} length {length}: over the bound by {over.max().item()}"
    if lse_row is not None:
        if length <= 0:
            assert (lse_row == -math.inf).all()
        else:
            vmax = max(b.c.rows(1, seq, range(length)).abs().max().item(), 1e-30)
            # the same score errors, plus the log's own rounding
            lim = (bound.max().item() / vmax) + 2.0**-21 * (lse.abs() + 1)
            if out_row.dtype == torch.bfloat16:
                lim = lim + 2.0**-8
            assert ((lse_row.double() - lse).abs() <= lim).all()


# ---- store and load -------------------------------------------------------------


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("heads,hd", [(5, 128), (2, 64), (3, 96), (1, 2), (2, 6), (1, 256), (2, 80), (7, 32)])
def test_store_codes_exact(cuda_backend, heads, hd, kv, rope, io):
    lens = [50, 1, 17]
    b = bench(cuda_backend, kv, heads, hd, lens, seed=3, fill="noise")
    before = b.c.pool.clone()
    g = torch.Generator(device=b.dev).manual_seed(hd + heads)
    rows = [(0, 49), (2, 0), (1, 0), (0, 3), (2, 16), (0, 31), (0, 32), (1, -1)]
    width = heads * hd
    x = torch.randn(len(rows), 3 * width + 5, device=b.dev, generator=g)
    x[3] = torch.randint(-9, 10, (x.shape[1],), device=b.dev, generator=g).float()  # ties
    x[4] = 0.25  # a constant row
    x[5] = 0.0
    x[6] *= 1e-41  # subnormal
    x = x.to(DT[io])
    k, v = x[:, 2:2 + width], x[:, 4 + width:4 + 2 * width]  # odd offsets and a wide stride
    cos = torch.randn(60, hd // 2, device=b.dev, generator=g)
    sin = torch.randn(60, hd // 2, device=b.dev, generator=g)
    b.store(k, v, [r[0] for r in rows], [r[1] for r in rows],
            rope=(cos.data_ptr(), sin.data_ptr(), 60) if rope else None)
    torch.cuda.synchronize()
    assert b.status.item() == 0
    kk, vv = k.double().view(-1, heads, hd), v.double().view(-1, heads, hd)
    if rope:
        p = torch.tensor([max(r[1], 0) for r in rows], device=b.dev)
        kk = R.rotate(kk, cos[p].double(), sin[p].double())
    want = R.Cache(kv, heads, hd, lens, b.dev, seed=3, fill="noise")
    for kind, val in ((0, kk), (1, vv)):
        c, s, z = R.quantise(kv, val)
        data = c.to(torch.int8).view(torch.uint8) if kv == KV_I8 else (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)
        for i, (seq, pos) in enumerate(rows):
            if pos < 0:
                continue
            page, slot = int(want.table[seq, pos // 16]), pos % 16
            want.codes_view(kind)[page, :, slot] = data[i]
            want.params_view(kind)[page, :, 0, slot] = s[i, :, 0].float()
            if kv == KV_I4:
                want.params_view(kind)[page, :, 1, slot] = z[i, :, 0].float()
    torch.testing.assert_close(b.c.pool, want.pool, rtol=0, atol=0)  # nothing else was written either
    assert not torch.equal(b.c.pool, before)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("heads,hd", [(5, 128), (2, 64), (1, 2), (2, 80), (1, 256), (3, 96)])
def test_load_values_exact(cuda_backend, heads, hd, kv, io):
    b = bench(cuda_backend, kv, heads, hd, [40, 5], seed=9)
    seq, pos = [0, 1, 0, 0, 1], [39, 4, 0, -1, 0]
    out = torch.full((5, 2 * heads * hd + 3), 5.0, device=b.dev, dtype=DT[io])
    k, v = out[:, 1:1 + heads * hd], out[:, 2 + heads * hd:2 + 2 * heads * hd]
    b.load(k, v, seq, pos)
    torch.cuda.synchronize()
    assert b.status.item() == 0
    for i in range(5):
        for kind, t in ((0, k), (1, v)):
            if pos[i] < 0:
                assert (t[i] == 5.0).all()
                continue
            want = b.c.rows(kind, seq[i], [pos[i]])[0].flatten().float().to(DT[io])
            torch.testing.assert_close(t[i], want, rtol=0, atol=0)
    assert (out[:, 0] == 5.0).all() and (out[:, 1 + heads * hd] == 5.0).all() and (out[:, -1] == 5.0).all()


@pytest.mark.parametrize("kv", KINDS)
def test_store_non_finite_and_bad_places(cuda_backend, kv):
    b = bench(cuda_backend, kv, 2, 64, [32], fill="zeros")
    k = torch.randn(4, 128, device=b.dev)
    v = torch.randn(4, 128, device=b.dev)
    k[1, 70] = float("nan")
    v[2, 3] = float("-inf")
    b.store(k, v, [0] * 4, [0, 1, 2, 3])
    torch.cuda.synchronize()
    assert b.status.item() == 1
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    b.load(ko, vo, [0] * 4, [0, 1, 2, 3])
    torch.cuda.synchronize()
    assert torch.isnan(ko[1, 64:]).all() and torch.isfinite(ko[1, :64]).all()
    assert torch.isnan(vo[2, :64]).all() and torch.isfinite(vo[2, 64:]).all()
    assert torch.isfinite(ko[[0, 2, 3]]).all()
    for seq, pos in ((1, 0), (-1, 0), (0, 32), (0, 10**9)):
        b.status.zero_()
        before = b.c.pool.clone()
        b.store(k[:1], v[:1], [seq], [pos])
        torch.cuda.synchronize()
        assert b.status.item() == 4 and torch.equal(b.c.pool, before)
    b.c.table[0, 1] = b.c.pages  # a page that is not there
    b.status.zero_()
    b.store(k[:1], v[:1], [0], [20])
    b.load(ko[:1], vo[:1], [0], [20])
    torch.cuda.synchronize()
    assert b.status.item() == 4


# ---- attention of single tokens ----------------------------------------------------


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("nh,heads,hd", [(20, 5, 128), (8, 2, 32), (16, 2, 64), (3, 3, 96), (12, 1, 128), (6, 2, 80),
                                         (5, 1, 256), (17, 1, 64), (2, 1, 2), (1, 1, 128), (24, 8, 64)])
def test_attention_lengths(cuda_backend, nh, heads, hd, kv, io):
    lens = [1, 0, 15, 16, 17, 130, 33, 700, 2]
    b = bench(cuda_backend, kv, heads, hd, lens, seed=hd)
    # the bytes behind each sequence's end may be anything
    for s, n in enumerate(lens):
        if n % 16:
            page = int(b.c.table[s, n // 16])
            for kind in (0, 1):
                b.c.params_view(kind)[page, :, :, n % 16:] = float("nan") if s % 2 else float("inf")
    g = torch.Generator(device=b.dev).manual_seed(1)
    q = torch.randn(len(lens), nh * hd + 3, device=b.dev, generator=g).to(DT[io])[:, 1:1 + nh * hd]
    out, lse = b.attend(q, nh, range(len(lens)), lens)
    assert b.status.item() == 0
    for i, n in enumerate(lens):
        check_row(b, q[i], nh, i, n, out[i], lse[i])


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("nh,heads,hd", [(20, 5, 128), (8, 1, 64), (4, 2, 32)])
@pytest.mark.parametrize("lens", [[9001], [5000, 1, 4999, 300, 0, 2048]])
def test_attention_split_and_joined(cuda_backend, lens, nh, heads, hd, kv):
    b = bench(cuda_backend, kv, heads, hd, lens, seed=5)
    q = 2 * torch.randn(len(lens), nh * hd, device=b.dev, generator=torch.Generator(device=b.dev).manual_seed(2))
    out, lse = b.attend(q, nh, range(len(lens)), lens, max_len=16 * b.c.per_seq)
    for i, n in enumerate(lens):
        check_row(b, q[i], nh, i, n, out[i], lse[i])
    again, lse2 = b.attend(q, nh, range(len(lens)), lens, max_len=16 * b.c.per_seq)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("kv", KINDS)
def test_attention_sharp_and_uneven_rows(cuda_backend, kv):
    """Scores far apart, values of very different size, a huge and a tiny q."""
    b = bench(cuda_backend, kv, 2, 128, [1000] * 4, seed=6)
    par = b.c.params_view(1)
    par[..., 0, ::3] *= 1e4  # some rows of V much larger
    par[..., 0, 1::3] *= 1e-4
    q = torch.randn(4, 8 * 128, device=b.dev, generator=torch.Generator(device=b.dev).manual_seed(3))
    q[0] *= 30
    q[1] *= 1e-30
    q[2] = 0
    q[3, :128] *= 1e4  # one head far above the others
    out, lse = b.attend(q, 8, range(4), [1000] * 4)
    for i in range(4):
        check_row(b, q[i], 8, i, 1000, out[i], lse[i])


def test_attention_rows_share_a_sequence_and_strides(cuda_backend):
    b = bench(cuda_backend, KV_I8, 2, 128, [333, 64], seed=7)
    big = torch.randn(5, 2 * 1024, device=b.dev)
    q = big[:, 512:512 + 1024]
    o = torch.full((5, 1500), 9.0, device=b.dev)
    seq, lens = [0, 0, 1, 0, 0], [333, 10, 64, 0, 200]
    out, _ = b.attend(q, 8, seq, lens, out=o[:, 300:300 + 1024], lse=False)
    for i in range(5):
        check_row(b, q[i], 8, seq[i], lens[i], out[i], None)
    assert (o[:, :300] == 9.0).all() and (o[:, 1324:] == 9.0).all()


@pytest.mark.parametrize("hd", [128, 32])
def test_attention_bad_places_are_reported(cuda_backend, hd):
    b = bench(cuda_backend, KV_I8, 1, hd, [100, 100], seed=8)
    q = torch.randn(3, 4 * hd, device=b.dev)
    out, _ = b.attend(q, 4, [0, 5, -1], [100, 10, 3])
    assert b.status.item() == 4
    check_row(b, q[0], 4, 0, 100, out[0], None)
    assert (out[1:] == 0).all()
    b.status.zero_()
    out, _ = b.attend(q[:1], 4, [0], [100], max_len=50)  # cut at max_len
    assert b.status.item() == 4
    check_row(b, q[0], 4, 0, 50, out[0], None)
    b.status.zero_()
    b.c.table[1, 3] = 10**6  # a page outside the pool is left out
    b.attend(q[:1], 4, [1], [100])
    assert b.status.item() == 4


@pytest.mark.parametrize("hd", [128, 32])
def test_attention_nan_is_not_hidden(cuda_backend, hd):
    b = bench(cuda_backend, KV_I8, 1, hd, [300], seed=8)
    b.c.params_view(0)[int(b.c.table[0, 2]), :, 0, 3] = float("nan")
    q = torch.randn(2, 4 * hd, device=b.dev)
    out, lse = b.attend(q, 4, [0, 0], [300, 30])
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all() and torch.isfinite(out[1]).all()
    q[1, hd + 1] = float("nan")  # one head of a row
    out, lse = b.attend(q, 4, [0, 0], [300, 30])
    assert torch.isnan(out[1, hd:2 * hd]).all() and torch.isfinite(out[1, :hd]).all()
    assert torch.isfinite(out[1, 2 * hd:]).all()


def test_attention_in_a_graph_and_on_another_stream(cuda_backend):
    lens = [700, 30, 1500, 1]
    b = bench(cuda_backend, KV_I4, 5, 128, lens, seed=4)
    nh = 20
    q = torch.randn(4, nh * 128, device=b.dev)
    seq, ln = b.ints(range(4)), b.ints(lens)
    want, _ = b.attend(q, nh, range(4), lens, max_len=1504)
    outs = [torch.zeros_like(q) for _ in range(2)]
    spaces = [b.space(nh) for _ in range(2)]
    side = torch.cuda.Stream(b.dev)
    graphs = []

    def call(i, stream):
        b.kv.attention(q.data_ptr(), outs[i].data_ptr(), 4, nh, seq.data_ptr(), ln.data_ptr(), 1504,
                       spaces[i].data_ptr(), spaces[i].numel(), b.status.data_ptr(), stream=stream)

    torch.cuda.synchronize()
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            call(i, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        other = torch.cuda.Stream(b.dev)
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o, want)
    # replayed with other lengths and queries
    ln.copy_(b.ints([3, 0, 1504, 1]))
    q.mul_(0.5)
    graphs[0].replay()
    torch.cuda.synchronize()
    for i, n in enumerate([3, 0, 1504, 1]):
        if n <= 16 * (-(-lens[i] // 16)):
            check_row(b, q[i], nh, i, n, outs[0][i], None)


# ---- attention of prompts --------------------------------------------------------


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("nh,heads,hd", [(20, 5, 128), (16, 2, 64), (4, 2, 32), (3, 3, 96), (9, 1, 128), (32, 8, 128),
                                         (32, 16, 64), (24, 8, 64), (40, 4, 128), (7, 7, 128)])
def test_prompt_attention(cuda_backend, nh, heads, hd, kv, io):
    counts, starts, seqs = [70, 0, 1, 33, 129], [0, 5, 40, 100, 17], [2, 0, 4, 1, 3]
    lens = [0] * 5
    for c, s, i in zip(counts, starts, seqs):
        lens[i] = c + s
    b = bench(cuda_backend, kv, heads, hd, lens, seed=hd + 1)
    cu = [3]  # rows before the first range and behind the last stay as they were
    for c in counts:
        cu.append(cu[-1] + c)
    q = torch.randn(cu[-1] + 4, nh * hd, device=b.dev, generator=torch.Generator(device=b.dev).manual_seed(5))
    q = q.to(DT[io])
    out, lse = b.prompt(q, nh, seqs, cu, starts)
    assert b.status.item() == 0
    assert (out[:3] == 77.0).all() and (out[cu[-1]:] == 77.0).all()
    assert (lse[:3] == 77.0).all() and (lse[cu[-1]:] == 77.0).all()
    for i, s in enumerate(seqs):
        for j in sorted({0, 1, 15, 16, 31, 32, 63, 64, counts[i] // 2, counts[i] - 2, counts[i] - 1}):
            if 0 <= j < counts[i]:
                r = cu[i] + j
                check_row(b, q[r], nh, s, starts[i] + j + 1, out[r], lse[r], fp16_weights=io == "bf16")


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("nh,heads,hd", [(20, 5, 128), (8, 2, 32)])
def test_prompt_attention_equals_single_rows(cuda_backend, nh, heads, hd, kv):
    """Every row of a long prompt, and of a few rows behind a long context, as the single-token operator has it."""
    counts, starts = [600, 5], [200, 4000]
    b = bench(cuda_backend, kv, heads, hd, [c + s for c, s in zip(counts, starts)], seed=3)
    q = torch.randn(605, nh * hd, device=b.dev, generator=torch.Generator(device=b.dev).manual_seed(5))
    out, lse = b.prompt(q, nh, [0, 1], [0, 600, 605], starts)
    seq = [0] * 600 + [1] * 5
    lens = [starts[0] + j + 1 for j in range(600)] + [starts[1] + j + 1 for j in range(5)]
    one, lse1 = b.attend(q, nh, seq, lens)
    # both are within the 32-bit bound of the same value (here about 1e-4 of max |v|)
    for i in (0, 300, 599, 600, 604):
        check_row(b, q[i], nh, seq[i], lens[i], out[i], lse[i])
        check_row(b, q[i], nh, seq[i], lens[i], one[i], lse1[i])
    bound = max(R.attention(b.c, q[i].double().view(nh, hd), seq[i], lens[i])[2].max().item()
                for i in (0, 150, 300, 450, 599, 602))
    assert (out - one).abs().max().item() <= 4 * bound


# ---- a run of them, as a decoder uses them ---------------------------------------------


@pytest.mark.parametrize("kv", KINDS)
def test_store_prompt_decode_run(cuda_backend, kv):
    """A prompt stored with RoPE and attended, then tokens one by one, against the same in 64 bits."""
    nh, heads, hd, n, steps = 8, 2, 128, 37, 6
    b = bench(cuda_backend, kv, heads, hd, [n + steps], fill="zeros")
    g = torch.Generator(device=b.dev).manual_seed(11)
    cos = torch.randn(64, hd // 2, device=b.dev, generator=g)
    sin = torch.randn(64, hd // 2, device=b.dev, generator=g)
    x = torch.randn(n + steps, (nh + 2 * heads) * hd, device=b.dev, generator=g)
    q, k, v = x.split([nh * hd, heads * hd, heads * hd], 1)
    rope = (cos.data_ptr(), sin.data_ptr(), 64)
    b.store(k[:n], v[:n], [0] * n, list(range(n)), rope)
    out, lse = b.prompt(q[:n], nh, [0], [0, n], [0])
    for i in range(n):
        check_row(b, q[i], nh, 0, i + 1, out[i], lse[i])
    for t in range(n, n + steps):
        b.store(k[t:t + 1], v[t:t + 1], [0], [t], rope)
        out, lse = b.attend(q[t:t + 1], nh, [0], [t + 1])
        check_row(b, q[t], nh, 0, t + 1, out[0], lse[0])
    p = torch.arange(n + steps, device=b.dev)
    kr = R.rotate(k.double().view(-1, heads, hd), cos[p].double(), sin[p].double())
    for kind, val in ((0, kr), (1, v.double().view(-1, heads, hd))):
        c, s, z = R.quantise(kv, val)
        assert torch.equal(b.c.rows(kind, 0, p), c.double() * s + z)
    assert b.status.item() == 0


# ---- the model's cache ------------------------------------------------------------------


@pytest.fixture(scope="module")
def small():
    cfg = ModelConfig(777, 512, 2, 4, 1, 640, 600, 10000.0, 1e-5)
    return cfg, synth.random_model(cfg, seed=5)


@pytest.fixture(scope="module")
def one_layer():
    """With one layer, K and V depend on the embedding alone, so the codes in the cache are the same however a prompt
    is cut into steps.  (With more, a last bit of an attention output can flip an int8 activation and that a 4-bit
    code of the next layer's V, a whole fifteenth of the row's range.)"""
    cfg = ModelConfig(777, 512, 1, 4, 1, 640, 600, 10000.0, 1e-5)
    return cfg, synth.random_model(cfg, seed=5)


def np_quantised(kv, x):
    c, s, z = R.quantise(kv, torch.from_numpy(np.ascontiguousarray(x)).double())
    return (c.double() * s + z).float().numpy()


@pytest.mark.parametrize("kv", KINDS)
def test_model_cache_write_read_fill(cuda_backend, small, kv):
    cfg, w = small
    m = BitNetModel(w, cuda_backend, max_batch_tokens=64)
    cache = m.new_kv_cache(num_pages=64, max_seqs=3, kv_dtype=kv)
    k, v = synth.kv_normal(3, 1, cfg, 45)
    cache.write(1, k, v)
    ko, vo = cache.read(1, 45)
    sh = (cfg.num_hidden_layers, 45, cfg.num_key_value_heads, cfg.head_dim())
    np.testing.assert_array_equal(ko.reshape(sh), np_quantised(kv, k.reshape(sh)))
    np.testing.assert_array_equal(vo.reshape(sh), np_quantised(kv, v.reshape(sh)))
    cache.fill_random(2, 33, 9)
    f32 = m.new_kv_cache(num_pages=64, max_seqs=3)
    f32.fill_random(2, 33, 9)
    sh = (cfg.num_hidden_layers, 33, cfg.num_key_value_heads, cfg.head_dim())
    for a, r in zip(cache.read(2, 33), f32.read(2, 33)):
        np.testing.assert_array_equal(a.reshape(sh), np_quantised(kv, r.reshape(sh)))
    k[0, 3, 5] = np.nan
    with pytest.raises(QuantizationError):
        cache.write(0, k, v)


@pytest.mark.parametrize("kv", KINDS)
def test_model_forward_over_a_quantised_cache(cuda_backend, one_layer, kv):
    """Prefill in one step, in chunks and token by token read the same codes.  Attention then differs by the order of
    32-bit sums, which can flip int8 roundings behind it: a flip moves one of 512 activations by 1/127 of the largest,
    some 1/(127 sqrt(512)) = 3.5e-4 of the result, so the 1e-2 of the tensor-core paths leaves room for tens of them.
    K and V are the quantised values of the f32 cache's."""
    cfg, w = one_layer
    m = BitNetModel(w, cuda_backend, max_batch_tokens=128)
    toks = synth.uniform_u32(12, 7, 100, 0, cfg.vocab_size - 1).tolist()
    full = m.new_kv_cache(num_pages=40, kv_dtype=kv)
    a = m.forward(toks, 0, full)
    assert m.attention_kernel(full, 1).startswith("kvq_attend")
    plain = m.new_kv_cache(num_pages=40)
    m.forward(toks, 0, plain)
    sh = (100, cfg.num_key_value_heads, cfg.head_dim())
    for x, y in zip(full.read(0, 100), plain.read(0, 100)):
        # K: f32 rotation in the f32 cache, 64-bit before quantising; codes may differ where that crosses a border
        r = np_quantised(kv, y[0].reshape(sh))
        step = (y[0].reshape(sh).max(-1) - y[0].reshape(sh).min(-1)).max() / (15 if kv == KV_I4 else 127)
        d = np.abs(x[0].reshape(sh) - r)
        assert d.max() <= 1.01 * step and np.mean(d > 1e-4 * step) < 1e-3
    one = m.new_kv_cache(num_pages=40, kv_dtype=kv)
    for i, t in enumerate(toks):
        b = m.forward([t], i, one)
    parts = m.new_kv_cache(num_pages=40, kv_dtype=kv)
    m.forward(toks[:33], 0, parts)
    c = m.forward(toks[33:], 33, parts)
    for other in (one, parts):
        for x, y in zip(full.read(0, 100), other.read(0, 100)):
            np.testing.assert_array_equal(x, y)
    assert np.max(np.abs(a - b)) <= 1e-2 * np.max(np.abs(a))
    assert np.max(np.abs(a - c)) <= 1e-2 * np.max(np.abs(a))


@pytest.mark.parametrize("kv", KINDS)
def test_model_decode_batch_and_layer_view(cuda_backend, small, kv):
    """A ragged batch through the captured decode graph, several steps, equal to the same steps launched one by one;
    the layer's view gives the operators the same cache."""
    cfg, w = small
    m = BitNetModel(w, cuda_backend, max_batch_tokens=64)
    lens = [1, 40, 300, 16, 511]
    cache = m.new_kv_cache(num_pages=80, max_seqs=len(lens), kv_dtype=kv)
    ref = m.new_kv_cache(num_pages=80, max_seqs=len(lens), kv_dtype=kv)
    for s, n in enumerate(lens):
        cache.fill_random(s, n, 21)
        ref.fill_random(s, n, 21)
    toks = [5, 6, 7, 8, 9]
    for _ in range(3):
        nxt, logits = m.decode_step(cache, range(len(lens)), toks, want_logits=True)
        n2, l2 = m.prefill(ref, range(len(lens)), [[t] for t in toks], want_logits=True)
        np.testing.assert_array_equal(logits, l2)
        np.testing.assert_array_equal(nxt, n2)
        toks = nxt.tolist()
    for s, n in enumerate(lens):
        for x, y in zip(cache.read(s, n + 3), ref.read(s, n + 3)):
            np.testing.assert_array_equal(x, y)
    dev = torch.device("cuda", cuda_backend.device_id)
    view = PagedKV.of_layer(cache, 1)
    k = torch.empty(30, cfg.kv_dim(), device=dev)
    v = torch.empty_like(k)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    seq = torch.full((30,), 2, dtype=torch.int32, device=dev)
    pos = torch.arange(30, dtype=torch.int32, device=dev)
    view.load(k.data_ptr(), v.data_ptr(), 30, seq.data_ptr(), pos.data_ptr(), st.data_ptr(), stream=1)
    torch.cuda.synchronize()
    kr, vr = cache.read(2, 30)
    np.testing.assert_array_equal(k.cpu().numpy(), kr[1])
    np.testing.assert_array_equal(v.cpu().numpy(), vr[1])
    with pytest.raises(InvalidConfig):
        PagedKV.of_layer(m.new_kv_cache(num_pages=4), 0)


@pytest.mark.parametrize("kv", KINDS)
def test_model_packed_prefill(cuda_backend, kv):
    """Ragged prompts packed into steps of 512 tokens run the prompt kernel (8 kv heads of 128), one of them split over
    steps; each sequence's logits against the same prompt by itself in steps of 16 (the single-token kernel).  One
    layer, so the codes are the same; the bound is that of test_model_forward_over_a_quantised_cache."""
    cfg = ModelConfig(300, 2048, 1, 16, 8, 256, 700, 10000.0, 1e-5)
    m = BitNetModel(synth.random_model(cfg, seed=3), cuda_backend, max_batch_tokens=512)
    prompts = [synth.uniform_u32(4, i, n, 0, 299).tolist() for i, n in enumerate([333, 1, 400, 60])]
    cache = m.new_kv_cache(num_pages=70, max_seqs=4, kv_dtype=kv)
    assert m.attention_kernel(cache, 512) == "kvq_prompt_kernel"
    _, logits = m.prefill_packed(cache, range(4), prompts, want_logits=True)
    ref = m.new_kv_cache(num_pages=70, max_seqs=4, kv_dtype=kv)
    for s, p in enumerate(prompts):
        for at in range(0, len(p), 16):
            r = m.forward(p[at:at + 16], at, ref, seq=s)
        for x, y in zip(cache.read(s, len(p)), ref.read(s, len(p))):
            np.testing.assert_array_equal(x, y)
        assert np.max(np.abs(logits[s] - r)) <= 1e-2 * np.max(np.abs(r))


@pytest.mark.parametrize("kv", KINDS)
def test_model_generate_runs(cuda_backend, small, kv):
    cfg, w = small
    m = BitNetModel(w, cuda_backend, max_batch_tokens=32)
    cache = m.new_kv_cache(num_pages=40, kv_dtype=kv)
    prompt = synth.uniform_u32(5, 9, 50, 0, cfg.vocab_size - 1).tolist()
    a = m.generate(cache, prompt, 20)
    b = m.generate(cache, prompt, 20)
    assert a == b and len(a) <= 20 and cache.len() == 50 + len(a)


def test_small_heads_run(cuda_backend):
    """Head sizes of the reference's unit-test model (4) and of 32."""
    from bitnetrs_b200 import tiny_config

    for cfg, w in ((tiny_config(), synth.tiny_reference_model(tiny_config())),
                   (ModelConfig(300, 256, 2, 8, 2, 384, 128, 500000.0, 1e-5),) * 2):
        if not hasattr(w, "layers"):
            w = synth.random_model(cfg, seed=4)
        m = BitNetModel(w, cuda_backend, max_batch_tokens=16)
        out = [m.forward([1, 2, 3], 0, m.new_kv_cache(num_pages=4, kv_dtype=kv)) for kv in (0, KV_I8)]
        assert np.max(np.abs(out[0] - out[1])) <= 0.2 * np.max(np.abs(out[0]))
    with pytest.raises((InvalidConfig, BackendError)):
        cfg = ModelConfig(64, 1024, 1, 2, 1, 64, 32, 10000.0, 1e-5)  # head_dim 512
        BitNetModel(synth.random_model(cfg, seed=4), cuda_backend, max_batch_tokens=4).new_kv_cache(4, kv_dtype=KV_I8)


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("hd", [128, 64, 32])
def test_prompt_attention_later_keys_stay_hidden(cuda_backend, hd, kv):
    """A key that is not a number, scale of K, of V or both, touches the rows that see it and no others; rows behind a
    negative start see nothing."""
    n = 200
    b = bench(cuda_backend, kv, 6, hd, [n, n], seed=2)
    for kind, pos in ((0, 150), (1, 70)):
        b.c.params_view(kind)[int(b.c.table[0, pos // 16]), 0, :, pos % 16] = float("nan")
    nh = 24  # the first four share the kv head in question
    q = torch.randn(2 * n, nh * hd, device=b.dev, generator=torch.Generator(device=b.dev).manual_seed(6))
    out, lse = b.prompt(q, nh, [0, 1], [0, n, 2 * n], [0, -40])
    o = out.view(2 * n, nh, hd)
    assert torch.isnan(o[70:n, :4]).all() and torch.isfinite(o[:n, 4:]).all() and torch.isfinite(o[:70]).all()
    assert torch.isnan(lse[150:n, :4]).all() and torch.isfinite(lse[:150]).all() and torch.isfinite(lse[:n, 4:]).all()
    for i in (0, 31, 69):
        check_row(b, q[i], nh, 0, i + 1, out[i], lse[i])
    assert (out[n:n + 40] == 0).all() and (lse[n:n + 40] == -math.inf).all()
    for i in (40, 41, 110, n - 1):
        check_row(b, q[n + i], nh, 1, i - 39, out[n + i], lse[n + i])


@pytest.mark.parametrize("hd", [128, 32])
def test_prompt_attention_bad_places_are_reported(cuda_backend, hd):
    nh = 48
    b = bench(cuda_backend, KV_I8, 12, hd, [100, 100], seed=8)
    q = torch.randn(100, nh * hd, device=b.dev)
    out, lse = b.prompt(q, nh, [0, 9], [0, 60, 100], [0, 5])
    assert b.status.item() == 4
    check_row(b, q[59], nh, 0, 60, out[59], lse[59])
    assert (out[60:] == 0).all() and (lse[60:] == -math.inf).all()
    b.status.zero_()
    out, lse = b.prompt(q, nh, [0], [0, 100], [0], max_len=50)  # cut there
    assert b.status.item() == 4
    check_row(b, q[49], nh, 0, 50, out[49], lse[49])
    check_row(b, q[80], nh, 0, 50, out[80], lse[80])
    b.status.zero_()
    b.c.table[1, 3] = 10**6
    b.prompt(q, nh, [1], [0, 100], [0])
    assert b.status.item() == 4


# ---- many rows, long sums, extremes, graphs ---------------------------------------------


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("hd", [32, 64, 96, 128, 256, 80])
def test_store_many_rows_as_few(cuda_backend, hd, kv, rope, io):
    """A store of many rows (more elements a lane) writes what stores of a few rows each write, which are tested above."""
    heads, n = 6, 1700
    one = bench(cuda_backend, kv, heads, hd, [n], seed=3, fill="noise")
    few = bench(cuda_backend, kv, heads, hd, [n], seed=3, fill="noise")
    g = torch.Generator(device=one.dev).manual_seed(hd)
    x = torch.randn(n, 2 * heads * hd, device=one.dev, generator=g)
    x[5] = torch.randint(-9, 10, (x.shape[1],), device=one.dev, generator=g).float()  # ties
    x[6] *= 1e-41
    x[7] = 0.25
    x[8, 3] = float("inf")
    k, v = x.to(DT[io]).split(heads * hd, 1)
    cos, sin = (torch.randn(n, hd // 2, device=one.dev, generator=g) for _ in range(2))
    angles = (cos.data_ptr(), sin.data_ptr(), n) if rope else None
    pos = torch.randperm(n, device=one.dev, generator=g).tolist()
    one.store(k, v, [0] * n, pos, angles)
    for i in range(0, n, 100):
        few.store(k[i:i + 100], v[i:i + 100], [0] * 100, pos[i:i + 100], angles)
    torch.cuda.synchronize()
    assert one.status.item() == few.status.item() == 1
    torch.testing.assert_close(one.c.pool, few.c.pool, rtol=0, atol=0)


def far(got, ref):
    return ((got.double() - ref).norm() / ref.norm()).item()


@pytest.mark.parametrize("shift", [0, 4, 8, 2])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("nh,heads,hd", [(32, 8, 128), (24, 12, 64)])
def test_long_sums_keep_their_accuracy(cuda_backend, nh, heads, hd, kv, shift):
    """f32 rows over long contexts, both kernels, with the output at every alignment of 4 bytes.

    Tensor cores cut their f32 sums.  Up to 64 such additions follow one another before a sum is added, rounded, to the
    rest: each cuts 2^-24 of the sum on average, and the sum is on average half of what it becomes, so a block is off
    by 64 * 2^-25 = 2^-19, and blocks, like their sums, add as independent terms.  The scores' 2 * hd / 16 additions
    and the weights' roundings are within 2^-20 together.  Below 2^-18.4 = 3e-6; a sum left in the tensor cores over
    1300 positions would be off by 5e-6 and more."""
    n, start = 90, 1250
    b = bench(cuda_backend, kv, heads, hd, [start + n, 700], seed=4)
    g = torch.Generator(device=b.dev).manual_seed(5)
    q = torch.randn(n + 600, nh * hd, device=b.dev, generator=g)
    wide = torch.full((n + 600, nh * hd + 12), 9.0, device=b.dev)
    out = wide[:, shift:shift + nh * hd] if shift != 8 else torch.zeros_like(q)
    a, c, s = b.ints([0, 1]), b.ints([0, n, n + 600]), b.ints([start, 100])
    sp, lse = b.space(nh), torch.zeros(n + 600, nh, device=b.dev)
    b.kv.prompt_attention(q.data_ptr(), out.data_ptr(), n + 600, nh, 2, a.data_ptr(), c.data_ptr(), s.data_ptr(),
                          start + n, sp.data_ptr(), sp.numel(), b.status.data_ptr(), ldo=out.stride(0),
                          lse=lse.data_ptr(), stream=1)
    torch.cuda.synchronize()
    assert b.status.item() == 0
    rows = [(0, 0, start + 1), (n // 2, 0, start + n // 2 + 1), (n - 1, 0, start + n), (n, 1, 101), (n + 410, 1, 511),
            (n + 411, 1, 512), (n + 412, 1, 513), (n + 599, 1, 700)]
    ref = []
    for r, seq, length in rows:
        check_row(b, q[r], nh, seq, length, out[r], lse[r])
        ref.append(R.attention(b.c, q[r].double().view(nh, hd), seq, length)[0].flatten())
    at = [r[0] for r in rows]
    assert far(out[at], torch.stack(ref)) < 3e-6
    one, _ = b.attend(q[at].contiguous(), nh, [r[1] for r in rows], [r[2] for r in rows])
    assert far(one, torch.stack(ref)) < 3e-6
    if shift != 8:
        assert (wide[:, :shift] == 9.0).all() and (wide[:, shift + nh * hd:] == 9.0).all()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("hd", [128, 64])
def test_prompt_attention_repeats_itself(cuda_backend, hd, kv, io):
    """A prompt of many more CTAs than the GPU holds, whose warps get in one another's way, gives the same bits every
    time, and every row what the single-token operator gives (bf16: within a weight's fp16 and the output's bf16)."""
    nh, heads, n = 32, 8, 2500
    b = bench(cuda_backend, kv, heads, hd, [n], seed=3)
    q = torch.randn(n, nh * hd, device=b.dev, generator=torch.Generator(device=b.dev).manual_seed(5)).to(DT[io])
    first, lse = b.prompt(q, nh, [0], [0, n], [0])
    for _ in range(25):
        again, lse2 = b.prompt(q, nh, [0], [0, n], [0])
        assert torch.equal(first, again) and torch.equal(lse, lse2)
    one, _ = b.attend(q, nh, [0] * n, list(range(1, n + 1)))
    # f32: both within 32-bit sums of the same, below 2^-15 of max |v|; bf16: a step of each output, and the weights' 2^-11
    vmax = b.c.rows(1, 0, list(range(n))).abs().max().item()
    off = (first.double() - one.double()).abs() - 2.0**-15 * vmax
    if io == "bf16":
        off = off - 2.0**-7 * one.double().abs() - 2.0**-11 * vmax
    assert (off <= 0).all()


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("hd", [128, 64, 32, 80])
def test_attention_of_large_keys_and_values(cuda_backend, hd, kv):
    """Keys near 2^72 under queries near 2^-72, values near 2^78: only powers of two against the ordinary case."""
    heads, nh, n = 8, 32, 300
    b = bench(cuda_backend, kv, heads, hd, [n], seed=12)
    b.c.params_view(0).mul_(2.0**72)
    b.c.params_view(1).mul_(2.0**78)
    q = torch.randn(n, nh * hd, device=b.dev, generator=torch.Generator(device=b.dev).manual_seed(1)) * 2.0**-72
    out, lse = b.prompt(q, nh, [0], [0, n], [0])
    one, lse1 = b.attend(q, nh, [0] * n, list(range(1, n + 1)))
    for i in (0, 77, 299):
        check_row(b, q[i], nh, 0, i + 1, out[i], lse[i])
        check_row(b, q[i], nh, 0, i + 1, one[i], lse1[i])


@pytest.mark.parametrize("kv", KINDS)
def test_store_prompt_load_in_a_graph(cuda_backend, kv):
    """A prompt's store, attention and read-back captured together and replayed for another prompt, shorter, of
    another sequence, with padding rows behind it."""
    heads, nh, hd, n = 8, 32, 128, 200
    b = bench(cuda_backend, kv, heads, hd, [n, n], fill="zeros")
    g = torch.Generator(device=b.dev).manual_seed(3)
    x = torch.randn(n, (nh + 2 * heads) * hd, device=b.dev, generator=g)
    q, k, v = x.split([nh * hd, heads * hd, heads * hd], 1)
    out, lse = torch.full((n, nh * hd), 7.0, device=b.dev), torch.full((n, nh), 7.0, device=b.dev)
    kb, vb = torch.full((n, heads * hd), 7.0, device=b.dev), torch.full((n, heads * hd), 7.0, device=b.dev)
    seq, pos = b.ints([0] * n), b.ints(range(n))
    run, cu, start = b.ints([0]), b.ints([0, n]), b.ints([0])
    sp = b.space(nh)

    def call(stream):
        b.kv.store(k.data_ptr(), v.data_ptr(), n, seq.data_ptr(), pos.data_ptr(), b.status.data_ptr(), ldk=x.stride(0),
                   ldv=x.stride(0), stream=stream)
        b.kv.prompt_attention(q.data_ptr(), out.data_ptr(), n, nh, 1, run.data_ptr(), cu.data_ptr(), start.data_ptr(),
                              n, sp.data_ptr(), sp.numel(), b.status.data_ptr(), ldq=x.stride(0), lse=lse.data_ptr(),
                              stream=stream)
        b.kv.load(kb.data_ptr(), vb.data_ptr(), n, seq.data_ptr(), pos.data_ptr(), b.status.data_ptr(), stream=stream)

    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream(b.dev)
    with torch.cuda.graph(graph, stream=side):
        call(torch.cuda.current_stream().cuda_stream)
    for s, m in ((0, n), (1, 133)):
        x.normal_(generator=g)
        for t in (out, lse, kb, vb):
            t.fill_(7.0)
        seq.fill_(s)
        pos[m:] = -1
        run.fill_(s)
        cu[1] = m
        graph.replay()
        torch.cuda.synchronize()
        assert b.status.item() == 0
        for i in (0, 63, 64, m - 1):
            check_row(b, q[i], nh, s, i + 1, out[i], lse[i])
        for kind, t in ((0, kb), (1, vb)):
            torch.testing.assert_close(t[:m], b.c.rows(kind, s, list(range(m))).flatten(1).float(), rtol=0, atol=0)
        for t in (out, lse, kb, vb):
            assert (t[m:] == 7.0).all()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("nh,heads,hd", [(32, 8, 32), (24, 12, 32), (24, 8, 96), (27, 9, 96), (36, 6, 96), (16, 16, 32)])
def test_prompt_attention_of_other_heads(cuda_backend, nh, heads, hd, kv, io):
    test_prompt_attention(cuda_backend, nh, heads, hd, kv, io)


@pytest.mark.parametrize("shift", [0, 8, 2])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("nh,heads,hd", [(24, 8, 96), (36, 12, 32)])
def test_long_sums_of_other_heads(cuda_backend, nh, heads, hd, kv, shift):
    test_long_sums_keep_their_accuracy(cuda_backend, nh, heads, hd, kv, shift)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("hd", [96, 32])
def test_prompt_attention_of_other_heads_repeats_itself(cuda_backend, hd, kv, io):
    test_prompt_attention_repeats_itself(cuda_backend, hd, kv, io)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("hd", [128, 64, 96, 32, 80])
def test_queries_and_outputs_at_odd_places(cuda_backend, hd, kv, io):
    """q and out that start on their element's size only, with odd row strides; both operators."""
    nh, heads, n = 24, 8, 150
    b = bench(cuda_backend, kv, heads, hd, [n], seed=6)
    g = torch.Generator(device=b.dev).manual_seed(2)
    big = torch.randn(n, nh * hd + 7, device=b.dev, generator=g).to(DT[io])
    q = big[:, 3:3 + nh * hd]
    wide = torch.full((n, nh * hd + 5), 9.0, device=b.dev, dtype=DT[io])
    out = wide[:, 1:1 + nh * hd]
    a, c, s, sp = b.ints([0]), b.ints([0, n]), b.ints([0]), b.space(nh)
    b.kv.prompt_attention(q.data_ptr(), out.data_ptr(), n, nh, 1, a.data_ptr(), c.data_ptr(), s.data_ptr(), n,
                          sp.data_ptr(), sp.numel(), b.status.data_ptr(), ldq=q.stride(0), ldo=out.stride(0),
                          bf16=io == "bf16", stream=1)
    torch.cuda.synchronize()
    for i in (0, 1, 63, 64, n - 1):
        check_row(b, q[i], nh, 0, i + 1, out[i], None, fp16_weights=io == "bf16")
    assert (wide[:, :1] == 9.0).all() and (wide[:, 1 + nh * hd:] == 9.0).all()
    wide.fill_(9.0)
    one, _ = b.attend(q[:9], nh, [0] * 9, [1, 2, 15, 16, 17, 100, n, 0, 33], out=out[:9], lse=False)
    for i, length in enumerate([1, 2, 15, 16, 17, 100, n, 0, 33]):
        check_row(b, q[i], nh, 0, length, one[i], None)
    assert b.status.item() == 0 and (wide[:, :1] == 9.0).all() and (wide[9:] == 9.0).all()


@pytest.mark.parametrize("hd", [128, 96, 80])
def test_nothing_to_attend_to(cuda_backend, hd):
    """Lengths of zero everywhere (max_len 0 too), prompts behind negative starts, no runs, empty runs, no rows."""
    nh, heads, n = 24, 8, 64
    b = bench(cuda_backend, KV_I8, heads, hd, [n, n], seed=6)
    q = torch.randn(n, nh * hd, device=b.dev)
    for most in (0, n, None):
        out, lse = b.attend(q, nh, [0, 1] * 32, [0] * n, max_len=most)
        assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = b.attend(q, nh, [0, 1] * 32, [-5] * n)
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = b.prompt(q, nh, [0], [0, n], [-n], max_len=0)
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = b.prompt(q, nh, [0, 1, 0], [5, 5, 5, 5], [0, 3, 9])
    assert (out == 77.0).all() and (lse == 77.0).all()
    out, lse = b.prompt(q, nh, [0, 1, 0, 1], [0, 0, 30, 30, 60], [0, 2, 9, 4])
    assert (out[60:] == 77.0).all() and b.status.item() == 0
    for r, seq, length in ((0, 1, 3), (29, 1, 32), (30, 1, 5), (59, 1, 34)):
        check_row(b, q[r], nh, seq, length, out[r], lse[r])
    assert b.attend(q[:0], nh, [], [])[0].shape[0] == 0


@pytest.mark.parametrize("kv,spare", [(KV_I8, 140000), (KV_I4, 260000)])
def test_pool_beyond_32_bits(cuda_backend, kv, spare):
    """Pages at more than 2^32 bytes into the pool: stored, read back and attended to."""
    nh, heads, hd, n = 32, 8, 128, 300
    b = bench(cuda_backend, kv, heads, hd, [n, 20], fill="zeros", spare=spare)
    assert b.c.pool.numel() > 2**32
    b.c.table[0] = b.c.pages - 1 - torch.arange(b.c.per_seq, dtype=torch.int32, device=b.dev)
    g = torch.Generator(device=b.dev).manual_seed(3)
    k, v = (torch.randn(n, heads * hd, device=b.dev, generator=g) for _ in range(2))
    q = torch.randn(n, nh * hd, device=b.dev, generator=g)
    b.store(k, v, [0] * n, list(range(n)))
    kb, vb = torch.zeros_like(k), torch.zeros_like(v)
    b.load(kb, vb, [0] * n, list(range(n)))
    out, lse = b.prompt(q, nh, [0], [0, n], [0])
    one, lse1 = b.attend(q, nh, [0] * n, list(range(1, n + 1)))
    assert b.status.item() == 0
    for kind, t in ((0, kb), (1, vb)):
        torch.testing.assert_close(t, b.c.rows(kind, 0, list(range(n))).flatten(1).float(), rtol=0, atol=0)
    assert kb.abs().amax(1).min() > 0
    for i in (0, 100, n - 1):
        check_row(b, q[i], nh, 0, i + 1, out[i], lse[i])
        check_row(b, q[i], nh, 0, i + 1, one[i], lse1[i])
