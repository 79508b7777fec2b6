"""The quantised paged key-value cache where its kernels can go wrong: values of very different size, weights that are
close to nothing, long sums, rows that are nearly constant, many runs, head sizes of the simple kernel.  Against the
64-bit forms of kvq_ref, as test_gpu_kvq."""
import numpy as np
import pytest

import kvq_ref as R
from bitnetrs_b200 import KV_I4, KV_I8, KV_BF16, BitNetModel, ModelConfig, synth
from test_gpu_kvq import DT, KINDS, bench, check_row, far

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def normal(b, seed, *shape):
    return torch.randn(*shape, device=b.dev, generator=torch.Generator(device=b.dev).manual_seed(seed))


def scale_rows(b, kind, seq, positions, factor):
    """Multiplies rows of the cache (all heads): their scales, and zeros, by `factor`."""
    for p in positions:
        b.c.params_view(kind)[int(b.c.table[seq, p // 16]), :, :, p % 16] *= factor


def put_row(b, kind, seq, pos, x):
    """Writes the quantised row x [hd] of f64 into all heads of one position."""
    code, s, z = R.quantise(b.c.kv, x)
    page, slot = int(b.c.table[seq, pos // 16]), pos % 16
    b.c.codes_view(kind)[page, :, slot] = (code.to(torch.int8).view(torch.uint8) if b.c.kv == KV_I8 else
                                           (code[0::2] | (code[1::2] << 4)).to(torch.uint8))
    b.c.params_view(kind)[page, :, 0, slot] = s.float()
    if b.c.kv == KV_I4:
        b.c.params_view(kind)[page, :, 1, slot] = z.float()


class Without:
    """A bench whose reference does not see some positions of the cache."""

    def __init__(self, b, skip):
        self.c, self.kv, self.kv_heads, self.hd, self.whole, self.skip = self, b.c.kv, b.c.kv_heads, b.c.hd, b.c, skip

    def rows(self, kind, seq, pos):
        return self.whole.rows(kind, seq, [int(p) for p in pos if int(p) not in self.skip])


# ---- values of very different size ------------------------------------------------------


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("hd", [128, 96, 64, 32])
@pytest.mark.parametrize("power", [20, 40, 70])
def test_prompt_rows_do_not_feel_the_size_of_later_values(cuda_backend, power, hd, kv, io):
    """Values 2^power times as large at positions 70 and 197 onwards: rows before them, in the same tile of keys and the
    same CTA, are as exact as without them (the bound counts the values that a row sees)."""
    n, heads, nh = 200, 8, 32
    b = bench(cuda_backend, kv, heads, hd, [n, n], seed=power)
    scale_rows(b, 1, 0, [70], 2.0**power)
    scale_rows(b, 1, 1, [197, 198, 199], 2.0**power)
    q = normal(b, 1, 2 * n, nh * hd).to(DT[io])
    out, lse = b.prompt(q, nh, [0, 1], [0, n, 2 * n], [0, 0])
    assert b.status.item() == 0
    for seq, rows in ((0, (0, 40, 63, 64, 65, 68, 69, 70, 71, 199)), (1, (0, 69, 128, 191, 192, 194, 196, 197, 199))):
        for i in rows:
            check_row(b, q[seq * n + i], nh, seq, i + 1, out[seq * n + i], lse[seq * n + i], fp16_weights=io == "bf16")


def far_below(b, seq, pos, power):
    """Makes position `pos` a key that every query with 4 in dimension 0 scores at most -4 * 1900 / sqrt(hd) < -470 (for
    hd <= 256), some 450 below the others, with values 2^power times as large: its weight is below 2^-600, so nothing
    of it may show in 32 bits, or in 64."""
    x = torch.zeros(b.c.hd, dtype=torch.float64, device=b.dev)
    x[0] = -2000
    put_row(b, 0, seq, pos, x)
    scale_rows(b, 1, seq, [pos], 2.0**power)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("hd", [128, 96, 64, 32])
@pytest.mark.parametrize("power", [30, 60])
def test_prompt_rows_do_not_feel_the_size_of_values_without_weight(cuda_backend, power, hd, kv, io):
    n, heads, nh = 200, 8, 32
    b = bench(cuda_backend, kv, heads, hd, [n], seed=power)
    skip = (3, 66, 150)
    for p in skip:
        far_below(b, 0, p, power)
    q = normal(b, 2, n, nh, hd)
    q[..., 0] = 4
    q = q.flatten(1).to(DT[io])
    out, lse = b.prompt(q, nh, [0], [0, n], [0])
    assert b.status.item() == 0
    for i in (2, 10, 63, 64, 70, 128, 149, 160, 199):
        left = i + 1
        check_row(Without(b, skip), q[i], nh, 0, left, out[i], lse[i], fp16_weights=io == "bf16")


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("nh,heads,hd", [(32, 8, 128), (8, 1, 128), (8, 2, 96), (16, 2, 64), (4, 2, 32), (6, 2, 80)])
@pytest.mark.parametrize("power", [30, 60])
def test_single_rows_do_not_feel_the_size_of_values_without_weight(cuda_backend, power, nh, heads, hd, kv, io):
    lens = [300, 20, 700, 5]
    b = bench(cuda_backend, kv, heads, hd, lens, seed=power + hd)
    skip = (3, 17, 250)
    for s, n in enumerate(lens):
        for p in skip:
            if p < n:
                far_below(b, s, p, power)
    q = normal(b, 3, len(lens), nh, hd)
    q[..., 0] = 4
    q = q.flatten(1).to(DT[io])
    for most in (700, 16 * b.c.per_seq):
        out, lse = b.attend(q, nh, range(len(lens)), lens, max_len=most)
        assert b.status.item() == 0
        for s, n in enumerate(lens):
            check_row(Without(b, skip), q[s], nh, s, n, out[s], lse[s])


@pytest.mark.parametrize("kv", KINDS)
def test_one_head_of_a_group_sees_large_values(cuda_backend, kv):
    """Heads that share a kv head, of which one alone gives its weight to a key with values 2^50 times as large."""
    hd, nh = 128, 4
    b = bench(cuda_backend, kv, 1, hd, [2000], seed=4)
    x = torch.zeros(hd, dtype=torch.float64, device=b.dev)
    x[0] = -2000
    put_row(b, 0, 0, 1000, x)
    scale_rows(b, 1, 0, [1000], 2.0**50)
    q = normal(b, 3, 1, nh, hd)
    q[..., 0] = 4
    q[:, 2, 0] = -4
    out, lse = b.attend(q.flatten(1), nh, [0], [2000])
    # its weight is 1, held to 2^-22; an I4 value's two parts and the five roundings on the way are below 2^-20 more
    v = b.c.rows(1, 0, [1000])[0, 0]
    assert ((out.view(nh, hd)[2].double() - v).abs() <= 2.0**-19 * v.abs().max()).all()
    one = Without(b, (1000,))
    ref, _, bound = R.attention(one, q[0].double(), 0, 2000)
    for h in (0, 1, 3):
        assert ((out.view(nh, hd)[h].double() - ref[h]).abs() <= bound[h]).all()


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [128, 96, 64, 32, 80])
@pytest.mark.parametrize("zero,scale", [(22, None), (30, None), (54, None), (78, None), (60, -60), (40, 0), (-90, None)])
def test_constant_and_nearly_constant_values(cuda_backend, zero, scale, hd, io):
    """I4 rows of V whose elements are all equal, near 2^zero: their scale is 0 and the zero holds them.  Or with a scale
    near 2^scale, far below the zero."""
    heads, nh, n = 8, 32, 200
    b = bench(cuda_backend, KV_I4, heads, hd, [n], seed=zero + 100)
    par = b.c.params_view(1)
    par[..., 1, :] = normal(b, 1, *par[..., 1, :].shape) * 2.0**zero
    par[..., 0, :] = 0.0 if scale is None else (1 + torch.rand(par[..., 0, :].shape, device=b.dev)) * 2.0**scale
    q = normal(b, 2, n, nh * hd).to(DT[io])
    out, lse = b.prompt(q, nh, [0], [0, n], [0])
    one, lse1 = b.attend(q, nh, [0] * n, list(range(1, n + 1)))
    assert b.status.item() == 0
    for i in (0, 1, 63, 64, 130, n - 1):
        check_row(b, q[i], nh, 0, i + 1, out[i], lse[i], fp16_weights=io == "bf16")
        check_row(b, q[i], nh, 0, i + 1, one[i], lse1[i])


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("hd", [128, 64])
def test_values_that_are_all_zero_at_first(cuda_backend, hd, kv):
    """The first 100 values are 0, the rest ordinary or near 2^-100."""
    heads, nh, n = 8, 32, 300
    for power in (0, -100):
        b = bench(cuda_backend, kv, heads, hd, [n], seed=5)
        b.c.params_view(1).mul_(2.0**power)
        scale_rows(b, 1, 0, range(100), 0.0)
        q = normal(b, 2, n, nh * hd)
        out, lse = b.prompt(q, nh, [0], [0, n], [0])
        one, lse1 = b.attend(q, nh, [0] * n, list(range(1, n + 1)))
        assert (out[:100] == 0).all() and (one[:100] == 0).all() and b.status.item() == 0
        for i in (100, 101, 127, 128, 200, 299):
            check_row(b, q[i], nh, 0, i + 1, out[i], None)
            check_row(b, q[i], nh, 0, i + 1, one[i], None)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("hd", [128, 64, 32, 80])
@pytest.mark.parametrize("at", [40, 64, 100])
def test_values_that_grow_far(cuda_backend, at, hd, kv, io):
    """Values near 2^-70 up to position `at`, near 2^75 from there on: the small ones no longer show in the output, but
    their weights still share it."""
    heads, nh, n = 8, 32, 200
    b = bench(cuda_backend, kv, heads, hd, [n], seed=9)
    scale_rows(b, 1, 0, range(at), 2.0**-70)
    scale_rows(b, 1, 0, range(at, n), 2.0**75)
    q = normal(b, 2, n, nh * hd).to(DT[io])
    out, lse = b.prompt(q, nh, [0], [0, n], [0])
    one, lse1 = b.attend(q, nh, [0] * n, list(range(1, n + 1)))
    assert b.status.item() == 0
    for i in (0, at - 1, at, at + 1, 127, 128, n - 1):
        check_row(b, q[i], nh, 0, i + 1, out[i], lse[i], fp16_weights=io == "bf16")
        check_row(b, q[i], nh, 0, i + 1, one[i], lse1[i])


# ---- long sums ----------------------------------------------------------------------------


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("nh,heads,hd", [(32, 8, 128), (64, 8, 128), (48, 12, 64), (16, 8, 32), (20, 10, 96)])
def test_long_sums_of_many_rows_keep_their_accuracy(cuda_backend, nh, heads, hd, kv):
    """So many rows that a warp of the single-token kernel has a whole context of 500 pages to itself.

    Tensor cores cut their f32 sums by 2^-24 of the sum on average at each addition, and a sum is on average half of
    what it becomes: 2^-25 a page.  At most 64 pages follow one another before a sum is added, rounded, to the rest, so a
    result is off by 2^-19, and its scores and weights within 2^-20: below 2^-18.4 = 3e-6.  Left in the tensor cores
    for 500 pages a sum would be off by 1.5e-5."""
    rows, n = 2400 // heads, 8000
    b = bench(cuda_backend, kv, heads, hd, [n], seed=4)
    q = normal(b, 5, rows, nh * hd)
    out, lse = b.attend(q, nh, [0] * rows, [n] * rows)
    assert b.status.item() == 0
    at = [0, 7, rows // 2, rows - 1]
    ref = []
    for r in at:
        check_row(b, q[r], nh, 0, n, out[r], lse[r])
        ref.append(R.attention(b.c, q[r].double().view(nh, hd), 0, n)[0].flatten())
    assert far(out[at], torch.stack(ref)) < 3e-6


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("nh,heads,hd", [(32, 8, 128), (24, 8, 96), (32, 8, 64), (32, 8, 32)])
def test_bf16_prompts_round_nothing_but_their_output(cuda_backend, nh, heads, hd, kv):
    """A bf16 output differs from the exact result's only where that lies next to the border of two bf16 values.

    With a result off by 3e-6 of the outputs' size r (the bound of the long sums), an output x is the other neighbour
    where the exact one is within 3e-6 r of a border.  Borders are 2^-8 to 2^-7 |x| apart, so that is a share of at most
    2 * 3e-6 * 2^8 E[min(r / |x|, 650)] of the outputs; for outputs spread like a normal the mean is at most 0.8 (1 +
    ln 650) = 6, the share 0.9 %.  A weight rounded to 11 bits moves results by some 2e-4 r: tens of per cent."""
    n = 512
    b = bench(cuda_backend, kv, heads, hd, [n], seed=3)
    q = normal(b, 5, n, nh * hd).to(torch.bfloat16)
    out, lse = b.prompt(q, nh, [0], [0, n], [0])
    rows = [63, 200, 333, 411, 470, n - 1]
    ref = []
    for r in rows:
        check_row(b, q[r], nh, 0, r + 1, out[r], lse[r])
        ref.append(R.attention(b.c, q[r].double().view(nh, hd), 0, r + 1)[0].flatten())
    same = out[rows].double() == torch.stack(ref).float().to(torch.bfloat16).double()
    assert (~same).double().mean().item() < 0.01


# ---- rows that are nearly constant ------------------------------------------------------------


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("heads,hd", [(6, 128), (6, 32), (6, 80), (6, 6)])
def test_store_of_rotated_rows_that_are_nearly_constant(cuda_backend, heads, hd, kv, many):
    """A rotated element is held in 64 bits and its row's zero in 32, so elements may lie below the zero: they are the
    least code.  Rows of a spread of 0 to 20 steps of 32 bits around 1.3 and 100, rotated by angles whose sine is 0."""
    n = 1700 if many else 80
    b = bench(cuda_backend, kv, heads, hd, [n], seed=3, fill="zeros")
    g = torch.Generator(device=b.dev).manual_seed(hd)
    base = torch.tensor([1.3, 100.0], device=b.dev).repeat(n // 2)[:, None, None]
    step = 2.0**-23 * torch.tensor([1.0, 64.0], device=b.dev).repeat(n // 2)[:, None, None]
    spread = torch.randint(0, 21, (n, heads, 1), device=b.dev, generator=g)
    k = base + step * torch.floor(torch.rand(n, heads, hd, device=b.dev, generator=g) * (spread + 1))
    k = k.flatten(1).contiguous()
    v = torch.randn(n, heads * hd, device=b.dev, generator=g)
    cos = (0.6 + 0.3 * torch.rand(n, 1, device=b.dev, generator=g)).repeat(1, hd // 2).contiguous()
    sin = torch.zeros(n, hd // 2, device=b.dev)
    b.store(k, v, [0] * n, list(range(n)), (cos.data_ptr(), sin.data_ptr(), n))
    torch.cuda.synchronize()
    assert b.status.item() == 0
    p = torch.arange(n, device=b.dev)
    kr = R.rotate(k.double().view(n, heads, hd), cos.double(), sin.double())
    below = kr.amin(-1) < kr.amin(-1).float().double()
    assert below.double().mean() > 0.2  # rows whose zero lies above their least element are among them
    for kind, val in ((0, kr), (1, v.double().view(n, heads, hd))):
        c, s, z = R.quantise(kv, val)
        page, slot = b.c.table[0, p // 16].long(), p % 16
        torch.testing.assert_close(b.c.params_view(kind)[page, :, 0, slot], s[..., 0].float(), rtol=0, atol=0)
        data = c.to(torch.int8).view(torch.uint8) if kv == KV_I8 else (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)
        torch.testing.assert_close(b.c.codes_view(kind)[page, :, slot], data, rtol=0, atol=0)


# ---- in a model ---------------------------------------------------------------------------------


def test_the_attention_kernel_of_decode_batches_is_named(cuda_backend):
    """As many tokens as the cache has sequences, or fewer, may be a decode step's, a token a sequence; more are a
    prompt's."""
    cfg = ModelConfig(300, 2048, 1, 16, 8, 256, 700, 10000.0, 1e-5)
    m = BitNetModel(synth.random_model(cfg, seed=3), cuda_backend, max_batch_tokens=512)
    for kv in KINDS:
        cache = m.new_kv_cache(num_pages=300, max_seqs=256, kv_dtype=kv)
        for tokens in (1, 2, 80, 256):
            assert m.attention_kernel(cache, tokens) == "kvq_attend_mma_kernel"
        for tokens in (257, 512):
            assert m.attention_kernel(cache, tokens) == "kvq_prompt_kernel"
        cache.close()


# ---- forms that no other test meets -----------------------------------------------------------------


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("hd", [128, 64])
def test_prompts_of_many_runs(cuda_backend, hd, kv, io):
    """More runs than a warp has lanes, empty ones among them."""
    heads, nh, runs = 8, 32, 75
    counts = [(7 * i) % 40 if i % 9 else 0 for i in range(runs)]
    starts = [(13 * i) % 90 for i in range(runs)]
    seqs = [(31 * i) % runs for i in range(runs)]
    lens = [0] * runs
    for c, s, i in zip(counts, starts, seqs):
        lens[i] = c + s
    b = bench(cuda_backend, kv, heads, hd, lens, seed=hd)
    cu = [0]
    for c in counts:
        cu.append(cu[-1] + c)
    q = normal(b, 5, cu[-1], nh * hd).to(DT[io])
    out, lse = b.prompt(q, nh, seqs, cu, starts)
    assert b.status.item() == 0 and (out != 77.0).all()
    for i in list(range(0, runs, 6)) + [31, 32, 33, 63, 64, 65, runs - 1]:
        for j in sorted({0, counts[i] // 2, counts[i] - 1}):
            if 0 <= j < counts[i]:
                check_row(b, q[cu[i] + j], nh, seqs[i], starts[i] + j + 1, out[cu[i] + j], lse[cu[i] + j],
                          fp16_weights=io == "bf16")


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("nh,heads,hd", [(8, 2, 100), (6, 3, 112), (4, 1, 256), (9, 1, 80)])
def test_other_head_sizes(cuda_backend, nh, heads, hd, kv, io):
    """Stored, read back and attended to with head sizes of the simple kernel, a prompt of 400 rows among them."""
    n = 400
    b = bench(cuda_backend, kv, heads, hd, [n, 77], fill="zeros")
    k, v, q = normal(b, 1, n, heads * hd), normal(b, 2, n, heads * hd), normal(b, 3, n, nh * hd).to(DT[io])
    b.store(k, v, [0] * n, list(range(n)))
    b.store(v[:77], k[:77], [1] * 77, list(range(77)))
    kb, vb = torch.zeros_like(k), torch.zeros_like(v)
    b.load(kb, vb, [0] * n, list(range(n)))
    out, lse = b.prompt(q, nh, [0], [0, n], [0])
    one, lse1 = b.attend(q[:3], nh, [1, 0, 1], [77, 399, 16])
    assert b.status.item() == 0
    for kind, x, back in ((0, k, kb), (1, v, vb)):
        c, s, z = R.quantise(kv, x.double().view(n, heads, hd))
        torch.testing.assert_close(back, (c.double() * s + z).flatten(1).float(), rtol=0, atol=0)
    for i in (0, 15, 16, 255, 330, n - 1):
        check_row(b, q[i], nh, 0, i + 1, out[i], lse[i])
    for i, (seq, length) in enumerate(((1, 77), (0, 399), (1, 16))):
        check_row(b, q[i], nh, seq, length, one[i], lse1[i])


@pytest.mark.parametrize("kv", KINDS)
def test_tensor_parallel_rank_over_a_quantised_cache(cuda_backend, kv):
    """The tensor-parallel form of the model's steps (a rank of one) over a quantised cache, bit for bit the plain one's."""
    from bitnetrs_b200 import tp

    cfg = ModelConfig(1000, 512, 2, 4, 2, 768, 256, 10000.0, 1e-5)
    w = synth.random_model(cfg, seed=21)
    prompts = [[(11 * i + 7 * j) % cfg.vocab_size for j in range(n)] for i, n in enumerate((5, 70, 9))]
    got = []
    for rank in (None, tp.TensorParallel(0, 1, tp.unique_id())):
        m = BitNetModel(w, cuda_backend, max_batch_tokens=128, tp=rank)
        cache = m.new_kv_cache(num_pages=64, max_seqs=3, kv_dtype=kv)
        nxt, logits = m.prefill(cache, [0, 1, 2], prompts, want_logits=True)
        got.append([logits, nxt])
        for _ in range(4):
            nxt, logits = m.decode_step(cache, [0, 1, 2], nxt, want_logits=True)
            got[-1] += [logits, nxt]
        got[-1] += list(cache.read(1, 74))
        cache.close()
        m.close()
    for a, b in zip(*got):
        np.testing.assert_array_equal(a, b)
