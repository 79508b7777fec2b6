"""The quantised key-value cache and the attention that reads it: cases, inputs, plain forms.

A page of the cache holds 16 positions.  A block is what one page holds of one
kv head: the K codes [16][head_dim], the V codes [16][head_dim], the K
parameters and the V parameters.  "i8" has codes in [-127, 127] and one scale a
row (value = code * scale); "i4" has codes in [0, 15], two to a byte (the even
dimension in the low half), and a scale and a zero a row (value = zero + code *
scale).  Scales and zeros are 32-bit floats, 16 of a kind together.

Four operators: `store` quantises rows of K and V into their slots (K rotated
first where the case has RoPE) and reads the same rows back; `load` reads rows
back alone; `attend` is attention of single tokens over their sequences;
`prompt` is causal attention of whole prompts, or parts of them, over theirs.
"""
import math
import random

import numpy as np
import torch

own = False

PAGE = 16
DEV = "cuda"
IO = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- cases ------------------------------------------------------------------


def listed():
    return [
        # the one new token of a single conversation, K rotated, heads of the 2B model
        {"name": "store-1-i8-rope", "op": "store", "kv": "i8", "io": "f32", "nh": 20, "nkv": 5, "hd": 128,
         "seqs": 1, "lo": 1, "hi": 1, "rope": True, "lens_seed": 1},
        # prompts of four users written at once, heads of the scaled model
        {"name": "store-prompts-i4", "op": "store", "kv": "i4", "io": "bf16", "nh": 32, "nkv": 8, "hd": 128,
         "seqs": 4, "lo": 1500, "hi": 2047, "rope": False, "lens_seed": 2},
        # a short conversation read back whole
        {"name": "load-517-i8", "op": "load", "kv": "i8", "io": "f32", "nh": 20, "nkv": 5, "hd": 128,
         "seqs": 1, "lo": 517, "hi": 517, "lens_seed": 3},
        # a batch's caches read back, as for another engine or a copy on disk
        {"name": "load-64-ragged-i4", "op": "load", "kv": "i4", "io": "bf16", "nh": 32, "nkv": 8, "hd": 128,
         "seqs": 64, "lo": 1, "hi": 4096, "lens_seed": 4},
        # the single-conversation decode step of the 2B model
        {"name": "attend-1x300-i8", "op": "attend", "kv": "i8", "io": "f32", "nh": 20, "nkv": 5, "hd": 128,
         "seqs": 1, "lo": 300, "hi": 300, "empty": 0, "lens_seed": 5},
        # one very long document, where the work has to be split over the length
        {"name": "attend-1x100003-i4", "op": "attend", "kv": "i4", "io": "bf16", "nh": 32, "nkv": 8, "hd": 128,
         "seqs": 1, "lo": 100003, "hi": 100003, "empty": 0, "lens_seed": 6},
        # the benchmark's decode batch: 256 sequences with contexts of 128 to 4096
        {"name": "attend-256-ragged-i8", "op": "attend", "kv": "i8", "io": "f32", "nh": 20, "nkv": 5, "hd": 128,
         "seqs": 256, "lo": 128, "hi": 4096, "empty": 0, "lens_seed": 7},
        # the scaled model's decode batch at a context of 2048
        {"name": "attend-64x2048-i4", "op": "attend", "kv": "i4", "io": "f32", "nh": 32, "nkv": 8, "hd": 128,
         "seqs": 64, "lo": 2048, "hi": 2048, "empty": 0, "lens_seed": 8},
        # eight heads to a kv head of 64, odd batch, some rows padding
        {"name": "attend-33-hd64-i8", "op": "attend", "kv": "i8", "io": "bf16", "nh": 16, "nkv": 2, "hd": 64,
         "seqs": 33, "lo": 1, "hi": 3001, "empty": 3, "lens_seed": 9},
        # a small model's heads of 32
        {"name": "attend-7-hd32-i4", "op": "attend", "kv": "i4", "io": "f32", "nh": 8, "nkv": 2, "hd": 32,
         "seqs": 7, "lo": 20, "hi": 700, "empty": 0, "lens_seed": 10},
        # one step of a packed prefill: 1024 tokens of a fresh prompt
        {"name": "prompt-1x1024-i8", "op": "prompt", "kv": "i8", "io": "f32", "nh": 20, "nkv": 5, "hd": 128,
         "seqs": 1, "lo": 1024, "hi": 1024, "before": 0, "lens_seed": 11},
        # prompts of odd lengths that go on from what their caches hold
        {"name": "prompt-4-ragged-i4", "op": "prompt", "kv": "i4", "io": "bf16", "nh": 32, "nkv": 8, "hd": 128,
         "seqs": 4, "lo": 301, "hi": 1501, "before": 1900, "lens_seed": 12},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "load", "attend", "attend", "prompt"])
    nkv = rng.choice([1, 2, 3, 5, 8])
    group = rng.choice([1, 2, 3, 4, 4, 5, 8])
    c = {"op": op, "kv": rng.choice(["i8", "i4"]), "io": rng.choice(["f32", "bf16"]), "nh": nkv * group, "nkv": nkv,
         "hd": rng.choice([32, 64, 64, 96, 128, 128, 128]), "lens_seed": rng.randrange(1 << 30)}
    if op in ("store", "load"):
        c["seqs"] = _log(rng, 1, 64)
        c["hi"] = _log(rng, 1, (6000 if op == "store" else 100000) // c["seqs"])
        c["lo"] = rng.randint(1, c["hi"])
        if op == "store":
            c["rope"] = rng.random() < 0.5
    elif op == "attend":
        c["seqs"] = _log(rng, 1, 200)
        c["hi"] = _log(rng, 1, min(80000, 400000 // c["seqs"]))
        c["lo"] = rng.randint(1, c["hi"])
        c["empty"] = rng.choice([0, 0, 1, c["seqs"] // 3])
    else:
        c["seqs"] = _log(rng, 1, 6)
        c["hi"] = _log(rng, 1, 2400 // c["seqs"])
        c["lo"] = rng.randint(1, c["hi"])
        c["before"] = rng.choice([0, _log(rng, 1, 2000)])
    return c


def _lengths(case):
    """Per sequence: new rows (store, load, prompt) or the context attended to (attend); and, for prompts, the
    positions that are there before.  A matter of the case alone."""
    rng = random.Random(case["lens_seed"])
    n = [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    for i in rng.sample(range(case["seqs"]), case.get("empty", 0)):
        n[i] = 0
    b = case.get("before", 0)
    before = [rng.randint(b // 2, b) for _ in n]
    if case["op"] == "store":
        before = [rng.randint(0, 3000) for _ in n]
    return n, before


def _row_bytes(case):
    return case["hd"] if case["kv"] == "i8" else case["hd"] // 2


def _block_bytes(case):
    return 2 * PAGE * _row_bytes(case) + (128 if case["kv"] == "i8" else 256)


def work(case):
    n, before = _lengths(case)
    nh, nkv, hd, eb = case["nh"], case["nkv"], case["hd"], 4 if case["io"] == "f32" else 2
    held = nkv * _block_bytes(case) / PAGE  # the cache's bytes for one position
    rows = sum(n)
    if case["op"] in ("store", "load"):
        x = rows * 2 * nkv * hd
        if case["op"] == "load":
            return {"bytes": rows * held + x * eb, "flops": 2 * x}
        return {"bytes": 2 * x * eb + rows * held + (rows * hd * 4 if case["rope"] else 0), "flops": 10 * x}
    if case["op"] == "attend":
        return {"bytes": rows * held + len(n) * nh * (2 * hd * eb + 4), "flops": 4 * nh * hd * rows}
    ctx = sum(a + b for a, b in zip(n, before))
    seen = sum(a * b + a * (a + 1) // 2 for a, b in zip(n, before))
    return {"bytes": ctx * held + rows * nh * (2 * hd * eb + 4), "flops": 4 * nh * hd * seen}


# ---- inputs -------------------------------------------------------------------


def _quantise(kv, x):
    """Codes, scales and zeros of rows x [..., hd] in 64 bits, where a value next to the border of two codes counts."""
    if kv == "i8":
        scale = (x.abs().amax(-1, keepdim=True) / 127).float()
        zero = torch.zeros_like(scale)
        least, most = -127, 127
    else:
        zero = x.amin(-1, keepdim=True).float()
        scale = ((x.amax(-1, keepdim=True) - zero.double()) / 15).float()
        least, most = 0, 15
    codes = torch.round((x - zero.double()) / scale.double().clamp_min(1e-300)).clamp(least, most)
    codes = torch.where(scale > 0, codes, torch.zeros_like(codes)).to(torch.int32)
    return codes, scale, zero


def _to_bytes(kv, codes):
    if kv == "i8":
        return codes.to(torch.int8).view(torch.uint8)
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def _to_codes(kv, data):
    if kv == "i8":
        return data.view(torch.int8).float()
    return torch.stack((data & 15, data >> 4), -1).flatten(-2).float()


def _regions(state, pool):
    """Views of blocks [..., block]: K codes, V codes [..., 16, row], and K and V parameters [..., kinds, 16]."""
    case = state["case"]
    row = _row_bytes(case)
    kinds = 1 if case["kv"] == "i8" else 2
    at = 2 * PAGE * row
    lead = pool.shape[:-1]
    k = pool[..., :PAGE * row].unflatten(-1, (PAGE, row))
    v = pool[..., PAGE * row:at].unflatten(-1, (PAGE, row))
    par = pool[..., at:].contiguous().view(torch.float32) if pool.shape != state["pool"].shape else \
        pool[..., at:].view(torch.float32)
    par = par.unflatten(-1, (2, kinds, PAGE))
    assert par.shape[:-3] == lead
    return k, v, par[..., 0, :, :], par[..., 1, :, :]


def _random_rows(gen, shape):
    """Keys and values as a model makes them: some channels much wider than others, rows of different size."""
    *lead, hd = shape
    wide = torch.exp(0.6 * torch.randn(hd, device=DEV, generator=gen))
    size = torch.exp(0.3 * torch.randn(*lead, 1, device=DEV, generator=gen))
    return torch.randn(*shape, device=DEV, generator=gen) * wide * size


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    n, before = _lengths(case)
    io, nh, nkv, hd, kv = IO[case["io"]], case["nh"], case["nkv"], case["hd"], case["kv"]
    total = [a + b for a, b in zip(n, before)] if case["op"] in ("store", "prompt") else n
    held = [-(-t // PAGE) for t in total]
    per_seq = max(max(held), 1)
    pages = sum(held) + 3
    order = torch.randperm(pages, device=DEV, generator=gen).to(torch.int32)
    table = torch.zeros(len(n), per_seq, dtype=torch.int32)
    filled = torch.arange(per_seq)[None, :] < torch.tensor(held)[:, None]
    table = table.to(DEV)
    table[filled.to(DEV)] = order[:sum(held)]
    pool = torch.empty(pages, nkv, _block_bytes(case), dtype=torch.uint8, device=DEV)
    state = {"case": case, "pool": pool, "table": table, "pages": pages, "per_seq": per_seq}
    k8, v8, kp, vp = _regions(state, pool)
    step = max(1, (1 << 25) // (nkv * PAGE * hd))
    for at in range(0, pages, step):
        end = min(pages, at + step)
        for codes, par in ((k8, kp), (v8, vp)):
            c, s, z = _quantise(kv, _random_rows(gen, (end - at, nkv, PAGE, hd)).double())
            codes[at:end] = _to_bytes(kv, c)
            par[at:end, :, 0] = s[..., 0]
            if kv == "i4":
                par[at:end, :, 1] = z[..., 0]
    seq = torch.repeat_interleave(torch.arange(len(n)), torch.tensor(n))
    first = torch.tensor(before)[seq]
    within = torch.arange(sum(n)) - torch.tensor([0] + n).cumsum(0)[:-1][seq]
    if case["op"] in ("store", "load"):
        pos = within + (first if case["op"] == "store" else 0)
        state |= {"rows": sum(n), "row_seq": seq.to(torch.int32).to(DEV), "row_pos": pos.to(torch.int32).to(DEV),
                  "k_out": torch.empty(sum(n), nkv * hd, dtype=io, device=DEV),
                  "v_out": torch.empty(sum(n), nkv * hd, dtype=io, device=DEV)}
    if case["op"] == "store":
        # the rows of a fused projection: [q | k | v]
        width = (nh + 2 * nkv) * hd
        qkv = torch.empty(sum(n), width, dtype=io, device=DEV)
        qkv[:, :nh * hd] = 0
        qkv[:, nh * hd:] = _random_rows(gen, (sum(n), 2 * nkv, hd)).flatten(1).to(io)
        state["k"], state["v"] = qkv[:, nh * hd:(nh + nkv) * hd], qkv[:, (nh + nkv) * hd:]
        state["rope_len"] = max(total)
        if case["rope"]:
            angle = torch.arange(max(total), dtype=torch.float64, device=DEV)[:, None] * \
                500000.0 ** (-torch.arange(hd // 2, dtype=torch.float64, device=DEV) * 2 / hd)
            state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    if case["op"] in ("attend", "prompt"):
        rows = len(n) if case["op"] == "attend" else sum(n)
        state["q"] = (1.3 * torch.randn(rows, nh, hd, device=DEV, generator=gen)).flatten(1).to(io)
        state |= {"rows": rows, "max_len": max(total), "out": torch.empty_like(state["q"]),
                  "lse": torch.empty(rows, nh, device=DEV)}
    if case["op"] == "attend":
        state["row_seq"] = torch.randperm(len(n), device=DEV, generator=gen).to(torch.int32)
        state["row_len"] = torch.tensor(n, dtype=torch.int32, device=DEV)[state["row_seq"].long()]
    if case["op"] == "prompt":
        state |= {"seq_ids": torch.arange(len(n), dtype=torch.int32, device=DEV),
                  "starts": torch.tensor(before, dtype=torch.int32, device=DEV),
                  "cu_rows": torch.tensor([0] + n, device=DEV).cumsum(0).to(torch.int32),
                  "most_rows": max(n), "row_seq": seq.to(DEV), "row_at": within.to(DEV)}
    return state


# ---- one pass -----------------------------------------------------------------


_backend = None


def _cache(state):
    """The framework's handle for the state's cache and the attention's workspace, made at the first pass and kept."""
    global _backend
    if "cache" not in state:
        import bitnetrs_b200 as b2
        if _backend is None:
            _backend = b2.CudaBackend(torch.cuda.current_device())
        case = state["case"]
        state["cache"] = b2.PagedKV(_backend, state["pool"].data_ptr(), state["table"].data_ptr(),
                                    pages=state["pages"], seqs=case["seqs"], pages_per_seq=state["per_seq"],
                                    kv_heads=case["nkv"], head_dim=case["hd"],
                                    kv_dtype=b2.KV_I8 if case["kv"] == "i8" else b2.KV_I4)
        state["status"] = torch.zeros(1, dtype=torch.int32, device=DEV)
        if case["op"] in ("attend", "prompt"):
            state["workspace"] = torch.empty(state["cache"].attention_workspace(case["nh"]), dtype=torch.uint8,
                                             device=DEV)
    return state["cache"]


def _run_own(state):
    case = state["case"]
    cache = _cache(state)
    # 1 is CUDA's name for the default stream that torch calls 0
    stream = torch.cuda.current_stream().cuda_stream or 1
    bf16 = case["io"] == "bf16"
    status = state["status"].data_ptr()
    if case["op"] in ("store", "load"):
        rows = (state["rows"], state["row_seq"].data_ptr(), state["row_pos"].data_ptr(), status)
        if case["op"] == "store":
            k, v = state["k"], state["v"]
            rope = (state["cos"].data_ptr(), state["sin"].data_ptr(), state["rope_len"]) if case["rope"] else None
            cache.store(k.data_ptr(), v.data_ptr(), *rows, ldk=k.stride(0), ldv=v.stride(0), bf16=bf16, rope=rope,
                        stream=stream)
        cache.load(state["k_out"].data_ptr(), state["v_out"].data_ptr(), *rows, bf16=bf16, stream=stream)
        return state["k_out"], state["v_out"]
    q, out, lse, space = state["q"], state["out"], state["lse"], state["workspace"]
    more = dict(bf16=bf16, lse=lse.data_ptr(), stream=stream)
    if case["op"] == "attend":
        cache.attention(q.data_ptr(), out.data_ptr(), state["rows"], case["nh"], state["row_seq"].data_ptr(),
                        state["row_len"].data_ptr(), state["max_len"], space.data_ptr(), space.numel(), status, **more)
    else:
        cache.prompt_attention(q.data_ptr(), out.data_ptr(), state["rows"], case["nh"], case["seqs"],
                               state["seq_ids"].data_ptr(), state["cu_rows"].data_ptr(), state["starts"].data_ptr(),
                               state["max_len"], space.data_ptr(), space.numel(), status, **more)
    return out, lse


def _values(state, data, par):
    """What codes [..., row] with parameters [..., kinds] stand for."""
    value = _to_codes(state["case"]["kv"], data) * par[..., :1]
    return value + par[..., 1:] if state["case"]["kv"] == "i4" else value


def _load(state):
    seq, pos = state["row_seq"].long(), state["row_pos"].long()
    page, slot = state["table"][seq, pos // PAGE].long(), pos % PAGE
    k8, v8, kp, vp = _regions(state, state["pool"])
    io = state["k_out"].dtype
    k = _values(state, k8[page, :, slot], kp[page, :, :, slot])
    v = _values(state, v8[page, :, slot], vp[page, :, :, slot])
    return k.flatten(1).to(io), v.flatten(1).to(io)


def _store(state):
    case = state["case"]
    seq, pos = state["row_seq"].long(), state["row_pos"].long()
    page, slot = state["table"][seq, pos // PAGE].long(), pos % PAGE
    k = state["k"].double().unflatten(1, (case["nkv"], case["hd"]))
    v = state["v"].double().unflatten(1, (case["nkv"], case["hd"]))
    if case["rope"]:
        cos, sin = state["cos"][pos].double()[:, None], state["sin"][pos].double()[:, None]
        lo, hi = k.chunk(2, -1)
        k = torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1)
    k8, v8, kp, vp = _regions(state, state["pool"])
    kc, ks, kz = _quantise(case["kv"], k)
    vc, vs, vz = _quantise(case["kv"], v)
    k8[page, :, slot] = _to_bytes(case["kv"], kc)
    v8[page, :, slot] = _to_bytes(case["kv"], vc)
    kinds = kp.shape[-2]
    kp[page, :, :, slot] = torch.cat((ks, kz), -1)[..., :kinds]
    vp[page, :, :, slot] = torch.cat((vs, vz), -1)[..., :kinds]
    return _load(state)


def _context(state, seq):
    """K and V of whole sequences, [seqs, kv heads, positions, hd] in 32 bits."""
    blocks = state["pool"][state["table"][seq].long()]
    k8, v8, kp, vp = _regions(state, blocks)
    # [seqs, pages, heads, kinds, 16] -> [..., 16, kinds]
    k = _values(state, k8, kp.transpose(-1, -2))
    v = _values(state, v8, vp.transpose(-1, -2))
    return k.transpose(1, 2).flatten(2, 3), v.transpose(1, 2).flatten(2, 3)


def _softmax_product(score, seen, v):
    """Softmax over the last axis where `seen`, times v; rows that see nothing give zeros.  And the log of the sum."""
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    return out, (top + torch.log(total)).squeeze(-1)


def _attend(state):
    case = state["case"]
    k, v = _context(state, state["row_seq"].long())
    q = state["q"].float().view(-1, case["nkv"], case["nh"] // case["nkv"], case["hd"])
    score = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(case["hd"])
    seen = torch.arange(k.shape[2], device=DEV) < state["row_len"][:, None]
    out, lse = _softmax_product(score, seen[:, None, None], v)
    return out.flatten(1).to(state["q"].dtype), lse.flatten(1)


def _prompt(state):
    case = state["case"]
    k, v = _context(state, state["seq_ids"].long())
    group = case["nh"] // case["nkv"]
    at = torch.arange(state["most_rows"], device=DEV)
    row = (state["cu_rows"][:-1, None] + at).clamp_max(state["rows"] - 1).long()
    q = state["q"].float()[row].view(case["seqs"], -1, case["nkv"], group, case["hd"]).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q, k[:, :, None].transpose(-1, -2)) / math.sqrt(case["hd"])
    seen = torch.arange(k.shape[2], device=DEV) <= (state["starts"][:, None] + at)[..., None]
    out, lse = _softmax_product(score, seen[:, None, None], v[:, :, None])
    out, lse = out.permute(0, 3, 1, 2, 4).flatten(2), lse.permute(0, 3, 1, 2).flatten(2)
    return out[state["row_seq"], state["row_at"]].to(state["q"].dtype), lse[state["row_seq"], state["row_at"]]


def run(state):
    if own:
        return _run_own(state)
    return {"store": _store, "load": _load, "attend": _attend, "prompt": _prompt}[state["case"]["op"]](state)


# ---- the definition in 64 bits ----------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    hd, nkv, group = case["hd"], case["nkv"], case["nh"] // case["nkv"]
    raw = state["pool"].view(-1)
    row = hd if case["kv"] == "i8" else hd // 2
    block = _block_bytes(case)

    def held(page, slot, kind):
        """K (0) or V (1) rows of pages [n] at slots [n], all heads, by byte addresses."""
        base = (page[:, None] * nkv + torch.arange(nkv, device=DEV)) * block
        d = torch.arange(hd, device=DEV)
        where = base + (kind * PAGE + slot[:, None]) * row
        if case["kv"] == "i8":
            code = raw[where[..., None] + d].to(torch.int64)
            code = torch.where(code > 127, code - 256, code)
        else:
            code = (raw[where[..., None] + d // 2].to(torch.int64) >> (4 * (d % 2))) & 15
        words = raw.view(torch.float32)
        each = 1 if case["kv"] == "i8" else 2
        p = (base + 2 * PAGE * row) // 4 + kind * each * PAGE + slot[:, None]
        x = code.double() * words[p].double()[..., None]
        return x if each == 1 else x + words[p + PAGE].double()[..., None]

    def place(seq, pos):
        return state["table"][seq, torch.div(pos, PAGE, rounding_mode="floor")].long(), pos % PAGE

    if case["op"] == "load":
        page, slot = place(state["row_seq"].long(), state["row_pos"].long())
        return held(page, slot, 0).flatten(1), held(page, slot, 1).flatten(1)
    if case["op"] == "store":
        both = []
        for x, turn in ((state["k"], case["rope"]), (state["v"], False)):
            x = x.double().reshape(-1, nkv, hd)
            if turn:
                p = state["row_pos"].long()
                z = torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * \
                    torch.complex(state["cos"][p].double(), state["sin"][p].double())[:, None]
                x = torch.cat((z.real, z.imag), -1)
            if case["kv"] == "i8":
                zero = torch.zeros_like(x[..., :1])
                scale = x.abs().max(-1, keepdim=True).values.div(127).float().double()
            else:
                zero = x.min(-1, keepdim=True).values.float().double()
                scale = (x.max(-1, keepdim=True).values - zero).div(15).float().double()
            both.append((zero + torch.round((x - zero) / scale) * scale).flatten(1))
        return tuple(both)
    outs, sums = [], []
    every = case["seqs"]
    for i in range(every):
        if case["op"] == "attend":
            seq, rows = int(state["row_seq"][i]), slice(i, i + 1)
            last = state["row_len"][i:i + 1].long() - 1
        else:
            seq, rows = i, slice(int(state["cu_rows"][i]), int(state["cu_rows"][i + 1]))
            last = int(state["starts"][i]) + torch.arange(rows.stop - rows.start, device=DEV)
        n = int(last.max()) + 1
        q = state["q"][rows].double().view(-1, nkv, group, hd)
        if n == 0:
            outs.append(torch.zeros_like(q).flatten(1))
            sums.append(torch.full((q.shape[0], nkv * group), -math.inf, dtype=torch.float64, device=DEV))
            continue
        pos = torch.arange(n, device=DEV)
        page, slot = place(torch.full_like(pos, seq), pos)
        k, v = held(page, slot, 0), held(page, slot, 1)
        score = torch.einsum("rhgd,phd->hgrp", q, k) / math.sqrt(hd)
        score = score.masked_fill(pos > last[:, None], -math.inf)
        lse = torch.logsumexp(score, -1)
        out = torch.einsum("hgrp,phd->rhgd", torch.exp(score - lse[..., None]), v)
        outs.append(out.flatten(1))
        sums.append(lse.permute(2, 0, 1).flatten(1))
    return torch.cat(outs), torch.cat(sums)
