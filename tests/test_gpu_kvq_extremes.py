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
