"""Refusals of the quantised-cache entry points, and the 64-bit reference itself: no GPU needed.  Addresses are never
followed: every call here is refused before a launch (the last one for want of a context)."""
import ctypes as C

import pytest

import kvq_ref as R
from bitnetrs_b200 import KV_I4, KV_I8, InvalidConfig, InvalidShape, PagedKV
from bitnetrs_b200 import _native as N

torch = pytest.importorskip("torch")
A = 1 << 20  # an aligned address that is never followed


def pages(**kw):
    d = dict(pool=A, page_table=A, pages=10, seqs=2, pages_per_seq=4, kv_heads=2, head_dim=64, kv_dtype=KV_I8)
    d.update(kw)
    return N.KvPages(*[d[f] for f, _ in N.KvPages._fields_])


def store(p, **kw):
    d = dict(k=A, ldk=128, v=A, ldv=128, bf16=0, rows=3, seq=A, pos=A, cos=None, sin=None, n=0, status=A)
    d.update(kw)
    N.check(N.cuda_lib().bitnet_cuda_kv_store_device(None, C.byref(p), *d.values(), None))


def load(p, **kw):
    d = dict(rows=3, seq=A, pos=A, k=A, ldk=128, v=A, ldv=128, bf16=0, status=A)
    d.update(kw)
    N.check(N.cuda_lib().bitnet_cuda_kv_load_device(None, C.byref(p), *d.values(), None))


def attend(p, **kw):
    d = dict(q=A, ldq=256, bf16=0, rows=3, nh=4, seq=A, lens=A, max_len=64, out=A, ldo=256, lse=None, space=A,
             bytes=1 << 30, status=A)
    d.update(kw)
    N.check(N.cuda_lib().bitnet_cuda_kv_attention_device(None, C.byref(p), *d.values(), None))


def prompt(p, **kw):
    d = dict(q=A, ldq=256, bf16=0, rows=3, nh=4, n=1, seqs=A, cu=A, starts=A, max_len=64, out=A, ldo=256, lse=None,
             space=A, bytes=1 << 30, status=A)
    d.update(kw)
    N.check(N.cuda_lib().bitnet_cuda_kv_prompt_attention_device(None, C.byref(p), *d.values(), None))


CALLS = [store, load, attend, prompt]


@pytest.mark.parametrize("call", CALLS)
def test_good_arguments_want_a_context(call):
    for p in (pages(), pages(kv_dtype=KV_I4), pages(head_dim=64)):
        with pytest.raises(InvalidShape) as e:
            call(p)
        assert e.value.expected == "non-null context"


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("bad,error", [
    (dict(pool=None), InvalidShape), (dict(pool=A + 8), InvalidShape), (dict(page_table=None), InvalidShape),
    (dict(page_table=A + 2), InvalidShape), (dict(pages=0), InvalidShape), (dict(seqs=0), InvalidShape),
    (dict(pages_per_seq=0), InvalidShape), (dict(kv_heads=0), InvalidShape), (dict(pages=1 << 31), InvalidShape),
    (dict(pages_per_seq=1 << 28), InvalidShape), (dict(head_dim=0), InvalidConfig), (dict(head_dim=63), InvalidConfig),
    (dict(head_dim=258), InvalidConfig), (dict(kv_dtype=1), InvalidConfig), (dict(kv_dtype=7), InvalidConfig)])
def test_bad_cache_is_refused(call, bad, error):
    with pytest.raises(error):
        call(pages(**bad))


@pytest.mark.parametrize("call,bad", [
    (store, dict(k=None)), (store, dict(v=A + 2)), (store, dict(ldk=127)), (store, dict(ldv=0)),
    (store, dict(seq=None)), (store, dict(pos=A + 1)), (store, dict(status=None)), (store, dict(cos=A)),
    (store, dict(sin=A, n=5)), (store, dict(cos=A, sin=A, n=0)), (store, dict(bf16=1, k=A + 1)),
    (store, dict(rows=1 << 30)),
    (load, dict(k=None)), (load, dict(v=A + 2)), (load, dict(ldk=127)), (load, dict(seq=None)),
    (load, dict(status=None)), (load, dict(rows=1 << 40)),
    (attend, dict(q=None)), (attend, dict(out=A + 2)), (attend, dict(ldq=255)), (attend, dict(ldo=1)),
    (attend, dict(nh=3)), (attend, dict(nh=0)), (attend, dict(max_len=65)), (attend, dict(space=None)),
    (attend, dict(space=A + 4)), (attend, dict(bytes=16)), (attend, dict(lse=A + 1)), (attend, dict(status=None)),
    (attend, dict(seq=None)), (attend, dict(lens=None)), (attend, dict(rows=1 << 31)),
    (prompt, dict(q=None)), (prompt, dict(nh=5)), (prompt, dict(seqs=None)), (prompt, dict(cu=None)),
    (prompt, dict(starts=A + 2)), (prompt, dict(max_len=1000)), (prompt, dict(bytes=0))])
def test_bad_arguments_are_refused(call, bad):
    with pytest.raises(InvalidShape) as e:
        call(pages(), **bad)
    assert e.value.expected != "non-null context"


def test_sizes():
    for kv in (KV_I8, KV_I4):
        for hd in (2, 64, 128, 256):
            assert PagedKV.block_bytes(kv, hd) == R.block_bytes(kv, hd) and R.block_bytes(kv, hd) % 16 == 0
    with pytest.raises(InvalidConfig):
        PagedKV.block_bytes(KV_I8, 3)
    with pytest.raises(InvalidConfig):
        PagedKV.block_bytes(1, 64)
    n = C.c_size_t()
    with pytest.raises(InvalidShape):
        N.check(N.cuda_lib().bitnet_cuda_kv_attention_workspace(C.byref(pages()), 3, C.byref(n)))
    N.check(N.cuda_lib().bitnet_cuda_kv_attention_workspace(C.byref(pages()), 8, C.byref(n)))
    assert n.value > 0


@pytest.mark.parametrize("kv", [KV_I8, KV_I4])
def test_reference_reads_what_it_writes(kv):
    g = torch.Generator().manual_seed(0)
    c = R.Cache(kv, 2, 32, [40], "cpu")
    x = torch.randn(c.pages, 2, 16, 32, dtype=torch.float64, generator=g)
    c.put_blocks(0, x)
    codes, s, z = R.quantise(kv, x)
    got = c.rows(0, 0, range(40))
    page = c.table[0, torch.arange(40) // 16].long()
    want = (codes.double() * s + z)[page, :, torch.arange(40) % 16]
    assert torch.equal(got, want)
    # a value is off by at most half a step, plus the rounding of scale and zero to 32 bits
    err = (codes.double() * s + z - x).abs()
    assert (err <= s * 0.5 + 2.0**-20 * x.abs().amax()).all()
