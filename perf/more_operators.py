"""Operators for long contexts that are read once or in part, as measurable
cases: attention of a batch that shares a prefix, and sparse attention over
selected cache blocks (the blocks' key bounds, the selection, the attention).

Each case is one pass as a serving engine makes it.  ``own`` chooses between
the package's entry points and a plain form of elementary torch operations:

- ``bounds``: the key bounds of the blocks that a step's new tokens touch,
              written and read back.
- ``select``: for each query row and KV head, the blocks whose bounds promise
              the largest scores.
- ``attend``: attention of each row over the blocks selected for it.
- ``layer``:  the three in a row, as one layer of a decode step runs them.
- ``prefix``: paged attention of a batch in which groups of sequences have
              their first keys in common.

Key bounds: of each block, for each KV head the int8 codes of every dim's least
key value (D bytes, rounded down) and largest (D bytes, rounded up), then one
exponent byte per KV head, padded to 16 bytes.  Codes stand for code x
2^(byte - 128), the least power of two, from 2^-100 on, at which the block's
largest magnitude is at most 127.  A query group is rounded (to even) to int8
by the same rule; a block's score is the largest, over the group's heads, of
the sums over dims of max(q lo, q hi): whole numbers times a power of two.

Lengths follow from the case alone, values and block tables from the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.float8_e4m3fn}
SIZES = {"f32": 4, "bf16": 2, "f16": 2, "fp8": 1}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # A busy 8B server's decode step: each sequence's newest block.
        _sparse("bounds_step_8b", "bounds", nd=64, lo=128, hi=4096),
        # Eight prompts: every block of them.
        _sparse("bounds_prompt_8b", "bounds", np=8, qlo=512, qhi=4096),
        # Decode far into long documents: 2,048 keys of up to 32,768 for each KV head.
        _sparse("select_step_8b", "select", nd=64, lo=8192, hi=32768, blocks=128),
        # One sequence of 130,001 keys: latency.
        _sparse("select_long_8b", "select", nd=1, lo=130001, hi=130001, blocks=256),
        # Two prompt chunks, each row with a selection of its own.
        _sparse("select_chunk_8b", "select", np=2, qlo=256, qhi=512, clo=8192, chi=16384, bs=32, blocks=64),
        # Eight chats of a 1B model: launch latency.
        _sparse("attend_step_1b", "attend", nd=8, lo=500, hi=8000, D=64, blocks=64),
        # Decode over the selected 2,048 keys.
        _sparse("attend_step_8b", "attend", nd=64, lo=4096, hi=32768, blocks=128),
        # Two prompt chunks over their rows' selections.
        _sparse("attend_chunk_8b", "attend", np=2, qlo=200, qhi=500, clo=8192, chi=16384, bs=32, blocks=64, dtype="f16"),
        # One layer of a long-context decode step, 70B heads, fp8 cache.
        _sparse("layer_70b_long", "layer", nd=32, lo=32768, hi=131072, Hq=64, bs=32, blocks=128, kv="fp8", first=1,
                recent=4),
        # Eight chats with one system prompt, 1B heads.
        _prefix("prefix_few_1b", groups=1, members=8, plo=2048, phi=2048, lo=16, hi=300, D=64),
        # A busy server with one long instruction: 8,192 keys in common.
        _prefix("prefix_step_8b", groups=1, members=64, plo=8192, phi=8192, lo=128, hi=2048),
        # Questions on four long documents, 70B heads: the largest call.
        _prefix("prefix_long_70b", groups=4, members=32, plo=16384, phi=32768, lo=128, hi=2048, Hq=64),
    ]


def _sparse(name, kind, nd=0, lo=0, hi=0, np=0, qlo=0, qhi=0, clo=0, chi=0, Hq=32, Hkv=8, D=128, dtype="bf16", kv=None,
            bs=16, blocks=64, first=1, recent=1):
    """``nd`` decode sequences of lo .. hi keys, ``np`` chunks of qlo .. qhi rows on clo .. chi cached keys."""
    return {"name": name, "kind": kind, "nd": nd, "lo": lo, "hi": hi, "np": np, "qlo": qlo, "qhi": qhi, "clo": clo,
            "chi": chi, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "kv": kv or dtype, "bs": bs, "blocks": blocks,
            "first": first, "recent": recent}


def _prefix(name, groups, members, plo, phi, lo, hi, alone=0, rows=1, Hq=32, Hkv=8, D=128, dtype="bf16", kv=None, bs=16):
    """``groups`` of ``members`` sequences with plo .. phi keys in common and lo .. hi of
    their own, ``rows`` of them queries, and ``alone`` sequences that share nothing."""
    return {"name": name, "kind": "prefix", "groups": groups, "members": members, "plo": plo, "phi": phi, "lo": lo,
            "hi": hi, "alone": alone, "rows": rows, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "kv": kv or dtype,
            "bs": bs}


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ones' ranges, sizes spread over them."""
    Hq, Hkv, D = rng.choice([(32, 8, 64), (32, 8, 128), (64, 8, 128)])
    bs = rng.choice([16, 16, 8, 32, 64, 24])
    kind = rng.choice(["bounds", "select", "select", "attend", "attend", "layer", "prefix", "prefix", "prefix"])
    if kind == "prefix":
        members = _logint(rng, 2, 96)
        plo = _logint(rng, 64, 16384)
        lo, rows = _logint(rng, 1, 512), rng.choice([1, 1, 1, 2])
        c = _prefix("", rng.choice([1, 1, 2, 3]), members, plo, plo * rng.choice([1, 2]), lo + rows, 4 * lo + rows,
                    rng.choice([0, 0, 1, 5]), rows, Hq, Hkv, D, rng.choice(["bf16", "bf16", "f16"]), None, bs)
        c["kv"] = rng.choice([c["dtype"], c["dtype"], "fp8"])
    else:
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        kv = rng.choice([dtype, dtype, "fp8"])
        first, recent = rng.choice([0, 1, 1, 2]), rng.choice([1, 1, 2, 5])
        blocks = first + recent + _logint(rng, 4, 4096 // bs)
        if rng.random() < 0.7:
            nd = _logint(rng, 1, 64)
            # at most half a million cached tokens
            lo = _logint(rng, 64, min(32768, (1 << 18) // nd))
            c = _sparse("", kind, nd=nd, lo=lo, hi=4 * lo)
        else:
            qlo, clo = _logint(rng, 8, 128), _logint(rng, 1, 8192)
            c = _sparse("", kind, np=rng.choice([1, 1, 2]), qlo=qlo, qhi=4 * qlo, clo=clo, chi=2 * clo)
        c.update(Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, kv=kv, bs=bs, blocks=blocks, first=first, recent=recent)
    del c["name"]
    return c


# ------------------------------------------------------------------ lengths
def _lengths(case):
    """(context lengths, query lengths) of a sparse batch."""
    g = torch.Generator().manual_seed(0)
    ctx = (torch.randint(case["lo"], case["hi"] + 1, (case["nd"],), generator=g) - 1).tolist()
    ql = [1] * case["nd"] + torch.randint(case["qlo"], case["qhi"] + 1, (case["np"],), generator=g).tolist()
    ctx += torch.randint(case["clo"], case["chi"] + 1, (case["np"],), generator=g).tolist()
    return ctx, ql


def _groups(case):
    """(lists of each group's sequences, keys in common, all lengths) of a prefix batch."""
    g = torch.Generator().manual_seed(0)
    n = case["groups"] * case["members"]
    P = torch.randint(case["plo"], case["phi"] + 1, (case["groups"],), generator=g).tolist()
    L = torch.randint(case["lo"], case["hi"] + 1, (n + case["alone"],), generator=g).tolist()
    order = torch.randperm(n + case["alone"], generator=g).tolist()      # an engine's slots are in no order
    seqs = [sorted(order[i * case["members"]:(i + 1) * case["members"]]) for i in range(case["groups"])]
    for s, p in zip(seqs, P):
        for i in s:
            L[i] += p
    return seqs, P, L


def _touched(case):
    """(sequence, block, keys in it) of the blocks that the step's new tokens reach."""
    bs, out = case["bs"], []
    for i, (c, n) in enumerate(zip(*_lengths(case))):
        out += [(i, b, min(bs, c + n - b * bs)) for b in range(c // bs, (c + n - 1) // bs + 1)]
    return out


def _record(case):
    return -(-case["Hkv"] * (2 * case["D"] + 1) // 16) * 16


# ------------------------------------------------------------------ inputs
class _Values:
    """N(0, 1) values drawn on the GPU from the seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def __call__(self, *shape, dtype):
        n, out = math.prod(shape), torch.empty(shape, dtype=dtype, device="cuda")
        flat = out.view(-1)
        for o in range(0, n, 1 << 26):
            m = min(1 << 26, n - o)
            flat[o:o + m] = torch.randn(m, generator=self.g, device="cuda").to(dtype)
        return out

    def keys(self, nb, case, dtype):
        """Keys of nb blocks: a block's have a mean in common, as neighbouring tokens do."""
        bs, Hkv, D = case["bs"], case["Hkv"], case["D"]
        out = torch.empty(nb, bs, Hkv, D, dtype=dtype, device="cuda")
        step = max(1, (1 << 26) // (bs * Hkv * D))
        for o in range(0, nb, step):
            m = min(step, nb - o)
            x = torch.randn(m, bs, Hkv, D, generator=self.g, device="cuda")
            x += torch.randn(m, 1, Hkv, D, generator=self.g, device="cuda")
            out[o:o + m] = x.to(dtype)
        return out.view(nb * bs, Hkv, D)

    def tables(self, need):
        """Block tables of sequences of `need` blocks; block 0 is the reserved one."""
        nb = sum(need) + 1
        perm = (torch.randperm(nb - 1, generator=self.g, device="cuda") + 1).to(torch.int32)
        bt = torch.zeros(len(need), max(need), dtype=torch.int32, device="cuda")
        o = 0
        for i, n in enumerate(need):
            bt[i, :n] = perm[o:o + n]
            o += n
        return nb, bt


def _sparse_inputs(case, seed):
    ctx, ql = _lengths(case)
    val = _Values(seed)
    Hq, Hkv, D, bs, dt, kv = case["Hq"], case["Hkv"], case["D"], case["bs"], DTYPES[case["dtype"]], DTYPES[case["kv"]]
    s = {"ctx": ctx, "ql": ql, "L": [c + q for c, q in zip(ctx, ql)]}
    nb, s["bt"] = val.tables([-(-x // bs) for x in s["L"]])
    R = sum(ql)
    s["seq"] = torch.repeat_interleave(torch.arange(len(ql)), torch.tensor(ql)).cuda()
    s["pos"] = torch.cat([torch.arange(c, c + n) for c, n in zip(ctx, ql)]).cuda()
    if case["kind"] != "bounds":
        s["q"] = val(R, Hq, D, dtype=dt)
    if case["kind"] != "select":
        s["k_cache"] = val.keys(nb, case, kv)
    if case["kind"] in ("attend", "layer"):
        s["v_cache"] = val(nb * bs, Hkv, D, dtype=kv)
        s["out"] = torch.empty_like(s["q"])
    if case["kind"] == "attend":
        s["selected"] = _any_selection(case, s, val.g)
    else:
        s["bounds"] = torch.zeros(nb, _record(case), dtype=torch.uint8, device="cuda")
    if case["kind"] == "select":
        # boxes of about the size that N(0, 1) keys of a block make
        c = torch.randn(nb, Hkv, D, generator=val.g, device="cuda") * 24
        r = 30 + 12 * torch.rand(nb, Hkv, D, generator=val.g, device="cuda")
        codes = torch.stack([(c - r).floor(), (c + r).ceil()], 2).clamp(-127, 127).to(torch.int8)
        s["bounds"][:, :Hkv * 2 * D] = codes.view(nb, -1).view(torch.uint8)
        e = torch.tensor([123] * 10 + [122, 124], dtype=torch.uint8, device="cuda")
        s["bounds"][:, Hkv * 2 * D:Hkv * 2 * D + Hkv] = e[torch.randint(0, 12, (nb, Hkv), generator=val.g, device="cuda")]
    if case["kind"] == "layer":           # the blocks of earlier steps
        k = s["k_cache"].view(nb, bs, Hkv, D)
        for o in range(0, nb, 4096):
            b = torch.arange(o, min(nb, o + 4096), device="cuda")
            _put_bounds(case, s["bounds"], b, k[o:o + 4096].to(torch.float32), torch.full_like(b, bs))
    s["touched"] = torch.tensor(_touched(case), dtype=torch.int64).cuda().t().contiguous()
    s["touched_blocks"] = s["bt"][s["touched"][0], s["touched"][1]].to(torch.int64)
    return s


def _any_selection(case, s, g):
    """A selection for each (row, KV head): the first and own block and others anywhere."""
    K, Hkv, bs = case["blocks"], case["Hkv"], case["bs"]
    R, width = len(s["pos"]), s["bt"].shape[1]
    last = (s["pos"] // bs)[:, None, None]
    sel = torch.empty(R, Hkv, K, dtype=torch.int32, device="cuda")
    for o in range(0, R, 256):
        b = torch.arange(width, device="cuda")
        u = torch.rand(len(last[o:o + 256]), Hkv, width, generator=g, device="cuda")
        lt = last[o:o + 256]
        u = torch.where((b < case["first"]) | (b > lt - case["recent"]), 2.0, u).masked_fill(b > lt, -1.0)
        top, at = u.topk(min(K, width), -1)
        at = at.masked_fill(top < 0, 1 << 30).sort(-1).values
        sel[o:o + 256] = -1
        sel[o:o + 256, :, :at.shape[-1]] = torch.where(at == 1 << 30, -1, at).to(torch.int32)
    return sel


def _prefix_inputs(case, seed):
    seqs, P, L = _groups(case)
    val = _Values(seed)
    Hq, Hkv, D, bs, kv = case["Hq"], case["Hkv"], case["D"], case["bs"], DTYPES[case["kv"]]
    # whole blocks of the common keys are held once; where the last is cut, each member has a copy
    whole = {i: p // bs for s, p in zip(seqs, P) for i in s}
    first = {i: s[0] for s in seqs for i in s}
    need = [-(-x // bs) for x in L]
    nb, bt = val.tables([n - (whole[i] if first.get(i, i) != i else 0) for i, n in enumerate(need)])
    full = torch.zeros(len(L), max(need), dtype=torch.int32, device="cuda")
    for i, n in enumerate(need):
        w = whole[i] if first.get(i, i) != i else 0
        full[i, w:n] = bt[i, :n - w]
        full[i, :w] = bt[first.get(i, i), :w]
    s = {"seqs": seqs, "P": P, "L": L, "bt": full, "q": val(case["rows"] * len(L), Hq, D, dtype=DTYPES[case["dtype"]])}
    for c in ("k_cache", "v_cache"):
        s[c] = val(nb * bs, Hkv, D, dtype=kv)
        pool = s[c].view(torch.uint8) if kv.itemsize == 1 else s[c]
        for m, p in zip(seqs, P):
            if p % bs:
                src = int(full[m[0], p // bs]) * bs
                for i in m[1:]:
                    dst = int(full[i, p // bs]) * bs
                    pool[dst:dst + p % bs] = pool[src:src + p % bs]
    s["out"] = torch.empty_like(s["q"])
    return s


def prepare(case, seed):
    """What the program holds before the call: inputs, and the plan of the engine step."""
    s = _prefix_inputs(case, seed) if case["kind"] == "prefix" else _sparse_inputs(case, seed)
    s["case"] = case
    if own:
        sizes = dict(num_q_heads=case["Hq"], num_kv_heads=case["Hkv"], head_dim=case["D"], block_size=case["bs"],
                     dtype=DTYPES[case["dtype"]], device="cuda")
        if case["kind"] == "prefix":
            from gllm_amd import paged
            s["plan"] = paged.AttentionPlan([case["rows"]] * len(s["L"]), s["L"],
                                            shared_prefixes=list(zip(s["seqs"], s["P"])), **sizes)
        else:
            from gllm_amd import sparse
            s["plan"] = sparse.SparsePlan(s["ql"], s["L"], blocks=case["blocks"], first_blocks=case["first"],
                                          recent_blocks=case["recent"], **sizes)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    kind, Hkv, D = case["kind"], case["Hkv"], case["D"]
    if kind == "prefix":
        if own:
            from gllm_amd import paged
            return paged.paged_attention(s["plan"], s["q"], s["k_cache"], s["v_cache"], s["bt"], out=s["out"])
        return _prefix_attention(case, s).to(s["q"].dtype)
    if own:
        from gllm_amd import sparse
        plan, res = s["plan"], []
        if kind in ("bounds", "layer"):
            sparse.write_key_bounds(plan, s["k_cache"], s["bounds"], s["bt"])
            res.append(sparse.key_bounds_values(s["bounds"], s["touched_blocks"], Hkv, D))
        sel = s.get("selected")
        if kind in ("select", "layer"):
            sel = sparse.select_blocks(plan, s["q"], s["bounds"], s["bt"])
            res.append(sel)
        if kind in ("attend", "layer"):
            res.append(sparse.sparse_attention(plan, s["q"], s["k_cache"], s["v_cache"], s["bt"], sel, out=s["out"]))
        return res
    res = []
    if kind in ("bounds", "layer"):
        _write_bounds(case, s)
        res.append(_get_bounds(case, s["bounds"], s["touched_blocks"]))
    sel = s.get("selected")
    if kind in ("select", "layer"):
        sel = _select(case, s)
        res.append(sel)
    if kind in ("attend", "layer"):
        res.append(_attend(case, s, sel).to(s["q"].dtype))
    return res


def _exponent(top):
    """Least e >= -100 with top <= 127 * 2^e, and whether it is at most 100."""
    m, e = torch.frexp(top)                               # top = m 2^e, 1/2 <= m < 1
    e = torch.where(m <= 127 / 128, e - 7, e - 6).clamp_min(-100)
    ok = torch.isfinite(top) & (e <= 100)
    return torch.where(ok, e, 0), ok


def _put_bounds(case, bounds, blocks, k, n):
    """Records of `blocks` from their first n keys k [blocks, bs, Hkv, D]."""
    Hkv, D = case["Hkv"], case["D"]
    there = torch.arange(k.shape[1], device=k.device)[None, :, None, None] < n[:, None, None, None]
    lo = k.masked_fill(~there, math.inf).amin(1)          # [blocks, Hkv, D]
    hi = k.masked_fill(~there, -math.inf).amax(1)
    e, ok = _exponent(torch.maximum(lo.abs(), hi.abs()).amax(-1))
    box = torch.stack([lo, hi], 2).to(torch.float64) * torch.exp2(-e.to(torch.float64))[..., None, None]
    box = torch.where(ok[..., None, None], box, 0)
    codes = torch.stack([box[:, :, 0].floor(), box[:, :, 1].ceil()], 2).to(torch.int8)
    w = Hkv * 2 * D
    bounds[blocks, :w] = codes.view(len(blocks), -1).view(torch.uint8)
    bounds[blocks, w:w + Hkv] = torch.where(ok, e + 128, 255).to(torch.uint8)


def _write_bounds(case, s):
    bs = case["bs"]
    n, blk = s["touched"][2], s["touched_blocks"]
    pool = s["k_cache"].view(-1, bs, case["Hkv"], case["D"])
    _put_bounds(case, s["bounds"], blk, (pool.view(torch.uint8)[blk].view(pool.dtype) if pool.dtype.itemsize == 1
                                         else pool[blk]).to(torch.float32), n)


def _get_bounds(case, bounds, blocks):
    """Bounds [blocks, Hkv, 2, D] as the values they stand for (infinities of an open block)."""
    Hkv, D = case["Hkv"], case["D"]
    rec = bounds[blocks]
    w = Hkv * 2 * D
    codes = rec[:, :w].contiguous().view(torch.int8).view(-1, Hkv, 2, D).to(torch.float32)
    e = rec[:, w:w + Hkv].to(torch.int32)
    x = codes * torch.exp2(e - 128.0)[..., None, None]
    open_ = torch.tensor([-math.inf, math.inf], device="cuda")[:, None]
    return torch.where((e == 255)[..., None, None], open_, x)


def _codes(q):
    """int8 codes (as fp32) of query groups [rows, Hkv, G, D]."""
    e, ok = _exponent(q.abs().amax((-1, -2)))
    return torch.where(ok[..., None, None], torch.round(q * torch.exp2(-e.to(torch.float32))[..., None, None]), 0)


def _select(case, s):
    Hkv, D, bs, K = (case[x] for x in ("Hkv", "D", "bs", "blocks"))
    G, R = case["Hq"] // Hkv, len(s["pos"])
    sel = torch.full((R, Hkv, K), -1, dtype=torch.int32, device="cuda")
    row = 0
    for i, n in enumerate(s["ql"]):
        for r0 in range(row, row + n, 256):
            r1 = min(row + n, r0 + 256)
            last = (s["pos"][r0:r1] // bs)[:, None, None]
            nb = -(-s["L"][i] // bs)
            rec = s["bounds"][s["bt"][i, :nb].to(torch.int64)]
            w = Hkv * 2 * D
            box = rec[:, :w].contiguous().view(torch.int8).view(nb, Hkv, 2 * D).to(torch.float32)
            c = _codes(s["q"][r0:r1].to(torch.float32).view(-1, Hkv, G, D))
            c = torch.cat([c.clamp_max(0), c.clamp_min(0)], -1)
            dots = torch.matmul(c.permute(1, 0, 2, 3).reshape(Hkv, -1, 2 * D), box.permute(1, 2, 0).contiguous())
            best = dots.view(Hkv, r1 - r0, G, nb).amax(2).permute(1, 0, 2)           # [rows, Hkv, nb]
            e = rec[:, w:w + Hkv].t().to(torch.float32)
            score = torch.where(e == 255, math.inf, best * torch.exp2(e - 128))
            b = torch.arange(nb, device="cuda")
            # blocks that are always taken come before all others, those behind the row after all
            rank = torch.where((b < case["first"]) | (b > last - case["recent"]), 2, torch.where(score == math.inf, 1, 0))
            rank = rank.masked_fill(b > last, -1)
            order = torch.sort(score.nan_to_num(posinf=0), dim=-1, descending=True, stable=True).indices
            order = order.gather(-1, torch.sort(rank.gather(-1, order), dim=-1, descending=True, stable=True).indices)
            k = min(K, nb)
            at = order[..., :k]
            at = at.masked_fill(rank.gather(-1, at) < 0, 1 << 30).sort(-1).values
            sel[r0:r1, :, :k] = torch.where(at == 1 << 30, -1, at).to(torch.int32)
        row += n
    return sel


def _rows(pool, slots, f):
    """pool[slot, h] for slots [rows, Hkv, n]."""
    h = torch.arange(pool.shape[1], device="cuda")[:, None]
    if pool.dtype.itemsize == 1:
        return pool.view(torch.uint8)[slots, h].view(pool.dtype).to(f)
    return pool[slots, h].to(f)


def _attend(case, s, sel):
    Hkv, D, bs, K = (case[x] for x in ("Hkv", "D", "bs", "blocks"))
    G, R, f = case["Hq"] // Hkv, len(s["pos"]), torch.float32
    out = torch.empty(s["q"].shape, dtype=f, device="cuda")
    step = max(1, (1 << 28) // (Hkv * K * bs * D))
    for r0 in range(0, R, step):
        b = sel[r0:r0 + step].to(torch.int64)                                        # [rows, Hkv, K]
        key = (b[..., None] * bs + torch.arange(bs, device="cuda"))
        seen = ((b[..., None] >= 0) & (key <= s["pos"][r0:r0 + step, None, None, None])).flatten(2)
        blk = s["bt"][s["seq"][r0:r0 + step, None, None], b.clamp_min(0)].to(torch.int64)
        slots = (blk[..., None] * bs + torch.arange(bs, device="cuda")).flatten(2)
        q = s["q"][r0:r0 + step].to(f).view(-1, Hkv, G, D)
        sc = torch.matmul(_rows(s["k_cache"], slots, f), q.transpose(-1, -2).contiguous()) / math.sqrt(D)
        sc = sc.masked_fill(~seen[..., None], -math.inf)                             # [rows, Hkv, keys, G]
        e = torch.exp(sc - sc.amax(-2, keepdim=True))
        p = (e / e.sum(-2, keepdim=True)).transpose(-1, -2).contiguous()
        out[r0:r0 + step] = torch.matmul(p, _rows(s["v_cache"], slots, f)).view(-1, Hkv * G, D)
    return out


def _prefix_attention(case, s):
    """softmax(q k^T / sqrt(D)) v of each sequence over all its keys."""
    Hkv, D, bs, n = (case[x] for x in ("Hkv", "D", "bs", "rows"))
    G, f = case["Hq"] // Hkv, torch.float32
    out = torch.empty(s["q"].shape, dtype=f, device="cuda")
    for i, L in enumerate(s["L"]):
        key = torch.arange(L, device="cuda")
        slot = s["bt"][i, key // bs].to(torch.int64) * bs + key % bs
        k, v = (_rows(s[c], slot.expand(1, Hkv, -1), f)[0] for c in ("k_cache", "v_cache"))   # [Hkv, L, D]
        q = s["q"][i * n:(i + 1) * n].to(f).view(n, Hkv, G, D).permute(1, 3, 0, 2).reshape(Hkv, D, n * G)
        sc = (torch.matmul(k, q.contiguous()) / math.sqrt(D)).view(Hkv, L, n, G)
        pos = L - n + torch.arange(n, device="cuda")
        sc = sc.masked_fill((key[:, None] > pos)[None, :, :, None], -math.inf)
        e = torch.exp(sc - sc.amax(1, keepdim=True))
        p = (e / e.sum(1, keepdim=True)).view(Hkv, L, n * G).transpose(1, 2).contiguous()
        out[i * n:(i + 1) * n] = torch.matmul(p, v).view(Hkv, n, G, D).permute(1, 0, 2, 3).reshape(n, Hkv * G, D)
    return out


# ------------------------------------------------------------------ work
def work(case):
    Hq, Hkv, D, bs = case["Hq"], case["Hkv"], case["D"], case["bs"]
    e, ekv = SIZES[case["dtype"]], SIZES[case["kv"]]
    if case["kind"] == "prefix":
        seqs, P, L = _groups(case)
        n = case["rows"]
        keys = sum(L) - sum((len(s) - 1) * p for s, p in zip(seqs, P))
        pairs = sum(n * x - n * (n - 1) // 2 for x in L)
        return {"bytes": keys * 2 * Hkv * D * ekv + 2 * n * len(L) * Hq * D * e + 4 * -(-keys // bs),
                "flops": 4 * Hq * D * pairs}
    ctx, ql = _lengths(case)
    K, nbytes, flops = case["blocks"], 0, 0
    rec = Hkv * (2 * D + 1)
    if case["kind"] in ("bounds", "layer"):               # the codes are written and read back
        t = _touched(case)
        nbytes += sum(x[2] for x in t) * Hkv * D * ekv + len(t) * (2 * rec + 4 + 8 + Hkv * 2 * D * 4)
        flops += 2 * sum(x[2] for x in t) * Hkv * D
    for c, n in zip(ctx, ql):
        nb = (np.arange(c, c + n) // bs + 1).astype(np.int64)
        if case["kind"] in ("select", "layer"):
            scored = nb[nb > K]
            nbytes += (int(nb.max()) * (rec + 4) if len(scored) else 0) + n * (Hq * D * e + Hkv * K * 4)
            flops += int(scored.sum()) * 4 * Hq * D
        if case["kind"] in ("attend", "layer"):
            # a row's own block is cut at its position
            keys = np.minimum(nb, K) * bs - (nb * bs - 1 - np.arange(c, c + n))
            nbytes += min(int(keys.sum()), c + n) * 2 * Hkv * D * ekv + n * (2 * Hq * D * e + Hkv * K * 4)
            flops += 4 * Hq * D * int(keys.sum())
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    if case["kind"] == "prefix":
        return _exact_prefix(case, _prefix_inputs(case, seed))
    s, res = _sparse_inputs(case, seed), []
    kind, Hkv, D, f = case["kind"], case["Hkv"], case["D"], torch.float64
    w = Hkv * 2 * D
    box = None
    if "bounds" in s:                                     # every block's box, as values
        e = s["bounds"][:, w:w + Hkv].to(f) - 128
        box = s["bounds"][:, :w].view(torch.int8).reshape(-1, Hkv, 2, D).to(f) * torch.exp2(e)[..., None, None]
    if kind in ("bounds", "layer"):
        for (i, b, n), blk in zip(_touched(case), s["touched_blocks"].tolist()):
            k = s["k_cache"][blk * case["bs"]:blk * case["bs"] + n].to(f)
            lo, hi = k.min(0).values, k.max(0).values
            top = torch.maximum(lo.abs(), hi.abs()).max(-1).values
            e = torch.floor(torch.log2(top.clamp_min(1e-300))) - 6
            e = torch.where(127 * torch.exp2(e) < top, e + 1, e)
            scale = torch.exp2(e.clamp_min(-100))[:, None]
            box[blk, :, 0], box[blk, :, 1] = torch.floor(lo / scale) * scale, torch.ceil(hi / scale) * scale
        res.append(box[s["touched_blocks"]])
    sel = s.get("selected")
    if kind in ("select", "layer"):
        sel = _exact_select(case, s, box)
        res.append(sel)
    if kind in ("attend", "layer"):
        out = torch.empty(s["q"].shape, dtype=f, device="cuda")
        G, bs, lists = case["Hq"] // Hkv, case["bs"], sel.cpu()
        for r, (i, p) in enumerate(zip(s["seq"].tolist(), s["pos"].tolist())):
            for h in range(Hkv):
                b = lists[r, h]
                key = (b[b >= 0].long()[:, None] * bs + torch.arange(bs)).flatten()
                key = key[key <= p].cuda()
                slot = s["bt"][i, key // bs].long() * bs + key % bs
                k, v = (s[c][:, h][slot].to(f) if s[c].dtype.itemsize > 1
                        else s[c].view(torch.uint8)[slot, h].view(s[c].dtype).to(f) for c in ("k_cache", "v_cache"))
                a = torch.softmax(s["q"][r, h * G:(h + 1) * G].to(f).mm(k.t().contiguous()) / math.sqrt(D), -1)
                out[r, h * G:(h + 1) * G] = a.mm(v)
        res.append(out)
    return res


def _exact_select(case, s, box):
    Hkv, D, bs, K = (case[x] for x in ("Hkv", "D", "bs", "blocks"))
    G, f, R = case["Hq"] // Hkv, torch.float64, len(s["pos"])
    sel = torch.full((R, Hkv, K), -1, dtype=torch.int32, device="cuda")
    for r, (i, p) in enumerate(zip(s["seq"].tolist(), s["pos"].tolist())):
        nb = p // bs + 1
        blk = s["bt"][i, :nb].long()
        for h in range(Hkv):
            if nb <= K:
                sel[r, h, :nb] = torch.arange(nb)
                continue
            q = s["q"][r, h * G:(h + 1) * G].to(f)
            top = q.abs().max()
            e = torch.floor(torch.log2(top.clamp_min(1e-300))) - 6
            e = torch.where(127 * torch.exp2(e) < top, e + 1, e).clamp_min(-100)
            c = torch.round(q / torch.exp2(e))
            lo, hi = box[blk, h, 0], box[blk, h, 1]                                    # [nb, D]
            score = torch.stack([torch.maximum(x * lo, x * hi).sum(-1) for x in c]).max(0).values
            forced = torch.zeros(nb, dtype=torch.bool, device="cuda")
            forced[:case["first"]] = True
            forced[nb - case["recent"]:] = True
            need = K - int(forced.sum())
            rest = score.masked_fill(forced, -math.inf)
            border = torch.sort(rest, descending=True).values[need - 1] if need else math.inf
            above = (rest > border) & ~forced
            tied = (rest == border) & ~forced
            tied &= tied.cumsum(0) <= need - above.sum()
            sel[r, h] = torch.nonzero(forced | above | tied)[:, 0].to(torch.int32)
    return sel


def _exact_prefix(case, s):
    Hkv, D, bs, n = (case[x] for x in ("Hkv", "D", "bs", "rows"))
    G, f = case["Hq"] // Hkv, torch.float64
    out = torch.empty(s["q"].shape, dtype=f, device="cuda")
    for i, L in enumerate(s["L"]):
        slots = (s["bt"][i, :-(-L // bs)].long()[:, None] * bs + torch.arange(bs, device="cuda")).flatten()[:L]
        k, v = (s[c][slots].to(f) if s[c].dtype.itemsize > 1 else s[c].view(torch.uint8)[slots].view(s[c].dtype).to(f)
                for c in ("k_cache", "v_cache"))
        hidden = torch.arange(L, device="cuda") > (L - n + torch.arange(n, device="cuda"))[:, None]
        for h in range(Hkv):
            q = s["q"][i * n:(i + 1) * n, h * G:(h + 1) * G].to(f)                     # [n, G, D]
            sc = q.reshape(n * G, D).mm(k[:, h].t().contiguous()).view(n, G, L) / math.sqrt(D)
            a = torch.softmax(sc.masked_fill(hidden[:, None], -math.inf), -1)
            out[i * n:(i + 1) * n, h * G:(h + 1) * G] = a.view(n * G, L).mm(v[:, h].contiguous()).view(n, G, D)
    return out
