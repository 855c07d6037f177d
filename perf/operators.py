"""The later operators of the attention path, as measurable cases: rotary
positions with the KV write, the 4-bit KV cache (write, read-back, attention)
and sliding-window attention with sink tokens.

Each case is one pass as a serving engine makes it.  ``own`` chooses between
the package's entry points and a plain form of elementary torch operations:

- ``rotary``: one layer's q and k rotated at their positions (pairs in halves
              or interleaved, part of the head, scaled frequencies) and k, v
              written to the paged cache.
- ``write4``: the same into a 4-bit cache, and the written rows read back.
- ``attn``:   paged attention of decode sequences and prompt chunks, over a
              4-bit cache, with a sliding window and sinks, or both.

The 4-bit cache: of each (block, KV head), ``bs`` rows of D / 2 code bytes
(e2m1, the even dim in the low half), then ``bs`` rows of D / 32 scale bytes
(2^(byte - 127)), padded to 16 bytes.  A block of 32 dims has the least
scale 2^e at which its largest magnitude rounds to 6 or less, |x| < 7 * 2^e.

Lengths follow from the case alone, values and block tables from the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.float8_e4m3fn}
SIZES = {"f32": 4, "bf16": 2, "f16": 2, "fp8": 1}
# positions scaled for long contexts, as model configurations give them
SCALING = {
    "none": None,
    "linear": {"rope_type": "linear", "factor": 4.0},
    "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
               "original_max_position_embeddings": 8192},
    "yarn": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # A decode step of eight chats, 1B heads: launch latency.
        _rotary("rotary_step_1b", n=8, Hq=32, Hkv=8, D=64, rot=64, scaling="llama3", pmax=131072),
        # The 19,679 prompt tokens of eight 8B prompts, interleaved pairs over
        # half of each head.
        _rotary("rotary_prompt_8b", n=19679, Hq=32, Hkv=8, D=128, rot=64, inter=True, scaling="yarn", pmax=32768),
        # A busy server's decode step into a 4-bit cache.
        _rotary("write4_step_8b", n=64, Hq=32, Hkv=8, D=128, rot=128, scaling="llama3", pmax=131072, kind="write4"),
        # Prompts into a 4-bit cache.
        _rotary("write4_prompt_8b", n=16384, Hq=32, Hkv=8, D=128, rot=128, scaling="llama3", pmax=32768,
                kind="write4"),
        # Four long chats decode together over a 4-bit cache.
        _attn("attn4_decode_8b_few", nd=4, lo=2048, hi=8192, kv="4"),
        # A busy 1B server's decode step over a 4-bit cache.
        _attn("attn4_decode_1b", nd=64, lo=128, hi=2048, Hq=32, Hkv=8, D=64, kv="4"),
        # Long-context decode, 70B heads, 4-bit cache: the largest call.
        _attn("attn4_decode_70b_long", nd=128, lo=16384, hi=32768, Hq=64, Hkv=8, D=128, kv="4"),
        # Continuous batching over a 4-bit cache: decodes and prompt chunks.
        _attn("attn4_mixed_8b", nd=128, lo=256, hi=8192, log=True, np=4, qlo=512, qhi=512, chi=4096, kv="4"),
        # Decode far past the window: 4,096 keys and four sinks of up to 32,768.
        _attn("window_decode_8b", nd=64, lo=4096, hi=32768, window=4096, sinks=4),
        # Prompt processing with a window of 1,024.
        _attn("window_prefill_8b", nd=0, np=8, qlo=512, qhi=8192, window=1024, sinks=4),
        # A small fp32 model's decode step with a window shorter than a block row.
        _attn("window_decode_f32", nd=8, lo=20, hi=2000, Hq=32, Hkv=8, D=64, dtype="f32", window=129, sinks=1),
        # Both: windowed decodes and chunks over a 4-bit cache.
        _attn("window4_mixed_8b", nd=64, lo=1024, hi=32768, log=True, np=2, qlo=256, qhi=1024, chi=8192, kv="4",
              window=2048, sinks=16),
    ]


def _rotary(name, n, Hq, Hkv, D, rot, pmax, inter=False, scaling="none", dtype="bf16", bs=16, kind="rotary"):
    return {"name": name, "kind": kind, "n": n, "Hq": Hq, "Hkv": Hkv, "D": D, "rot": rot, "inter": inter,
            "scaling": scaling, "theta": 500000.0, "pmax": pmax, "dtype": dtype, "bs": bs}


def _attn(name, nd, lo=0, hi=0, np=0, qlo=0, qhi=0, chi=0, Hq=32, Hkv=8, D=128, dtype="bf16", kv=None, bs=16,
          log=False, window=0, sinks=0):
    """``window`` 0: every earlier key; ``kv`` "4": the 4-bit cache."""
    return {"name": name, "kind": "attn", "nd": nd, "lo": lo, "hi": hi, "log": log, "np": np, "qlo": qlo, "qhi": qhi,
            "chi": chi, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "kv": kv or dtype, "bs": bs, "window": window,
            "sinks": sinks}


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ones' ranges, sizes spread over them."""
    Hq, Hkv, D = rng.choice([(32, 8, 64), (32, 8, 128), (64, 8, 128)])
    bs = rng.choice([16, 16, 8, 32, 24])
    f16 = rng.choice(["bf16", "bf16", "f16"])
    kind = rng.choice(["rotary", "write4", "attn4", "attn4", "window", "window", "window_f32"])
    if kind in ("rotary", "write4"):
        rot = rng.choice([D, D, D // 2, D // 4])
        c = _rotary("", _logint(rng, 1, 16384), Hq, Hkv, D, rot, rng.choice([8192, 131072, 1048576]),
                    rng.choice([False, True]), rng.choice(list(SCALING)), rng.choice([f16, f16, "f32"]), bs, kind)
    elif kind == "window_f32":
        lo = _logint(rng, 16, 1024)
        Dg = rng.choice([64, 64, 96, 128])
        c = _attn("", _logint(rng, 1, 16), lo, 4 * lo, rng.choice([0, 0, 1]), 16, 128, 512, 32, 8, Dg, "f32",
                  None, bs, window=_logint(rng, 8, 1024), sinks=rng.choice([0, 1, 4, 17]))
    else:
        window, sinks, kv = 0, 0, "4"
        if kind == "window":
            window, sinks = _logint(rng, 16, 8192), rng.choice([0, 0, 1, 4, 64])
            kv = rng.choice([None, None, "fp8", "4"])
        shape = rng.choice(["decode", "decode", "prefill", "mixed"])
        if shape == "decode":
            lo = _logint(rng, 64, 8192)
            # at most a quarter million cached tokens
            nd = _logint(rng, 1, max(1, min(256, (1 << 18) // (2 * lo))))
            c = _attn("", nd, lo, 3 * lo, 0, 0, 0, 0, Hq, Hkv, D, f16, kv, bs, window=window, sinks=sinks)
        elif shape == "prefill":
            qlo = _logint(rng, 16, 1024)
            c = _attn("", 0, 0, 0, _logint(rng, 1, 8), qlo, 4 * qlo, rng.choice([0, 0, 1024]), Hq, Hkv, D, f16, kv,
                      bs, window=window, sinks=sinks)
        else:
            lo, qlo = _logint(rng, 64, 1024), _logint(rng, 16, 512)
            c = _attn("", _logint(rng, 8, 64), lo, 8 * lo, _logint(rng, 1, 4), qlo, 2 * qlo, 2048, Hq, Hkv, D, f16,
                      kv, bs, log=True, window=window, sinks=sinks)
    del c["name"]
    return c


# ------------------------------------------------------------------ lengths
def _lengths(case):
    """(context lengths, query lengths) of an attention batch."""
    g = torch.Generator().manual_seed(0)
    nd, lo, hi = case["nd"], case["lo"], case["hi"]
    if case["log"]:
        u = torch.rand(nd, generator=g, dtype=torch.float64).tolist()
        L = [int(round(math.exp(math.log(lo) + x * (math.log(hi) - math.log(lo))))) for x in u]
    else:
        L = torch.randint(lo, hi + 1, (nd,), generator=g).tolist()
    ctx, ql = [x - 1 for x in L], [1] * nd
    if case["np"]:
        ql += torch.randint(case["qlo"], case["qhi"] + 1, (case["np"],), generator=g).tolist()
        ctx += torch.randint(0, case["chi"] + 1, (case["np"],), generator=g).tolist()
    return ctx, ql


def _first(case, ctx):
    """First key inside the window of the row at position ctx."""
    return max(0, ctx + 1 - case["window"]) if case["window"] else 0


def _frequencies(case, f):
    """(rotation per position of each pair, factor of cos and sin) from the
    model configuration, in 64 bits."""
    R, theta, sc = case["rot"], case["theta"], SCALING[case["scaling"]]
    i = torch.arange(R // 2, dtype=f)
    base = theta ** (-2 * i / R)
    if sc is None:
        return base, 1.0
    factor = sc["factor"]
    if sc["rope_type"] == "linear":
        return base / factor, 1.0
    orig = sc["original_max_position_embeddings"]
    if sc["rope_type"] == "llama3":
        # turns made over the original length: few turns are slowed down, many are kept
        turns = orig * base / (2 * math.pi)
        lo, hi = sc["low_freq_factor"], sc["high_freq_factor"]
        keep = ((turns - lo) / (hi - lo)).clamp(0, 1)
        return base * (keep + (1 - keep) / factor), 1.0
    # yarn: pairs that make more than 32 turns are kept, fewer than one slowed down

    def dim(n):
        return R * math.log(orig / (n * 2 * math.pi)) / (2 * math.log(theta))
    lo, hi = max(math.floor(dim(32)), 0), min(math.ceil(dim(1)), R - 1)
    keep = 1 - ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return base * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1


# ------------------------------------------------------------------ inputs
class _Values:
    """N(0, 1) values, and the bytes of a 4-bit cache of such values, drawn on
    the GPU from the seed."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def __call__(self, *shape, dtype):
        n, out = math.prod(shape), torch.empty(shape, dtype=dtype, device="cuda")
        flat = out.view(-1)
        for o in range(0, n, 1 << 26):
            m = min(1 << 26, n - o)
            flat[o:o + m] = torch.randn(m, generator=self.g, device="cuda").to(dtype)
        return out

    def _bytes(self, n, table):
        out = torch.empty(n, dtype=torch.uint8, device="cuda")
        for o in range(0, n, 1 << 26):
            m = min(1 << 26, n - o)
            r = torch.randint(0, table.numel(), (m,), generator=self.g, device="cuda", dtype=torch.int32)
            out[o:o + m] = table[r]
        return out

    def pool4(self, nb, Hkv, bs, D):
        # 256 quantiles of N(0, 1) as codes at scale 1/2; their pairs make a byte
        x = torch.erfinv((torch.arange(256, dtype=torch.float64) + 0.5) / 128 - 1) * math.sqrt(2) / 0.5
        a = x.abs()
        code = sum((a > t).to(torch.int64) for t in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)) + 8 * (x < 0)
        pairs = (code[:, None] * 16 + code[None, :]).reshape(-1).to(torch.uint8).cuda()
        scales = torch.tensor([126] * 13 + [125, 127, 127], dtype=torch.uint8).cuda()
        pool = torch.zeros(nb, Hkv, _record(bs, D), dtype=torch.uint8, device="cuda")
        pool[..., :bs * D // 2] = self._bytes(nb * Hkv * bs * D // 2, pairs).view(nb, Hkv, -1)
        pool[..., bs * D // 2:bs * D // 32 * 17] = self._bytes(nb * Hkv * bs * D // 32, scales).view(nb, Hkv, -1)
        return pool


def _record(bs, D):
    return -(-(bs * D // 32 * 17) // 16) * 16


def _rotary_inputs(case, seed):
    val = _Values(seed)
    n, Hq, Hkv, D, bs, dt = case["n"], case["Hq"], case["Hkv"], case["D"], case["bs"], DTYPES[case["dtype"]]
    s = {"q": val(n, Hq, D, dtype=dt), "k": val(n, Hkv, D, dtype=dt), "v": val(n, Hkv, D, dtype=dt)}
    if n < 256:               # a decode step: every token at its own position
        s["pos"] = torch.randint(0, case["pmax"], (n,), generator=val.g, device="cuda")
    else:                     # prompts, one after another
        s["pos"] = torch.arange(n, device="cuda") % case["pmax"]
    nb = -(-n // bs) + 1
    s["slots"] = (torch.randperm((nb - 1) * bs, generator=val.g, device="cuda") + bs)[:n].contiguous()
    for c in ("k_cache", "v_cache"):
        s[c] = torch.zeros(nb, Hkv, _record(bs, D), dtype=torch.uint8, device="cuda") if case["kind"] == "write4" \
            else torch.zeros(nb * bs, Hkv, D, dtype=dt, device="cuda")
    s["q_out"] = torch.empty_like(s["q"])
    return s


def _attn_inputs(case, seed):
    ctx, ql = _lengths(case)
    L = [c + q for c, q in zip(ctx, ql)]
    Hq, Hkv, D, bs = case["Hq"], case["Hkv"], case["D"], case["bs"]
    val = _Values(seed)
    need = [-(-x // bs) for x in L]
    nb = sum(need) + 1                                    # block 0 is the reserved one
    perm = (torch.randperm(nb - 1, generator=val.g, device="cuda") + 1).to(torch.int32)
    bt = torch.zeros(len(L), max(need), dtype=torch.int32, device="cuda")
    o = 0
    for i, n in enumerate(need):
        bt[i, :n] = perm[o:o + n]
        o += n
    s = {"ctx": ctx, "ql": ql, "L": L, "bt": bt, "q": val(sum(ql), Hq, D, dtype=DTYPES[case["dtype"]])}
    for c in ("k_cache", "v_cache"):
        s[c] = val.pool4(nb, Hkv, bs, D) if case["kv"] == "4" else val(nb * bs, Hkv, D, dtype=DTYPES[case["kv"]])
    s["out"] = torch.empty_like(s["q"])
    return s


def prepare(case, seed):
    """What the program holds before the call: inputs, the model's rotary
    positions, and the plan of the engine step."""
    if case["kind"] != "attn":
        s = _rotary_inputs(case, seed)
        f, m = _frequencies(case, torch.float64)
        s["freq"], s["factor"] = f.cuda(), m
        if own:
            import gllm_amd
            s["rotary"] = gllm_amd.Rotary(case["D"], theta=case["theta"], rotary_dim=case["rot"],
                                          interleaved=case["inter"], scaling=SCALING[case["scaling"]], device="cuda")
    else:
        s = _attn_inputs(case, seed)
        if own:
            from gllm_amd import paged
            s["plan"] = paged.AttentionPlan(s["ql"], s["L"], num_q_heads=case["Hq"], num_kv_heads=case["Hkv"],
                                            head_dim=case["D"], block_size=case["bs"], dtype=s["q"].dtype,
                                            device="cuda", window=case["window"] or None, sinks=case["sinks"])
    s["case"] = case
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if case["kind"] == "attn":
        if own:
            from gllm_amd import paged
            return paged.paged_attention(s["plan"], s["q"], s["k_cache"], s["v_cache"], s["bt"], out=s["out"])
        return _attention(case, s, torch.float32).to(s["q"].dtype)
    if own:
        from gllm_amd import paged
        paged.rotary_kv_write(s["k"], s["v"], s["pos"], s["rotary"], s["k_cache"], s["v_cache"], s["slots"],
                              q=s["q"], q_out=s["q_out"])
        if case["kind"] == "rotary":
            return s["q_out"], s["k_cache"], s["v_cache"]
        return (s["q_out"],) + tuple(paged.kv4_values(s[c], s["slots"], case["D"], s["q"].dtype)
                                     for c in ("k_cache", "v_cache"))
    # angles of far positions need 64 bits; so do rows that are rounded to
    # 4 bits, where they come next to a border
    ang = s["pos"].to(torch.float64)[:, None] * s["freq"]
    c, sn = torch.cos(ang) * s["factor"], torch.sin(ang) * s["factor"]
    c32, s32 = c.to(torch.float32), sn.to(torch.float32)
    dt = s["q"].dtype
    s["q_out"].copy_(_rotate(case, s["q"].to(torch.float32), c32, s32).to(dt))
    if case["kind"] == "rotary":
        s["k_cache"][s["slots"]] = _rotate(case, s["k"].to(torch.float32), c32, s32).to(dt)
        s["v_cache"][s["slots"]] = s["v"]
        return s["q_out"], s["k_cache"], s["v_cache"]
    for name, x in (("k_cache", _rotate(case, s["k"].to(torch.float64), c, sn)), ("v_cache", s["v"].to(torch.float32))):
        _put4(case, s[name], s["slots"], x)
    return (s["q_out"],) + tuple(_get4(case, s[n], s["slots"], torch.float32).to(dt) for n in ("k_cache", "v_cache"))


def _rotate(case, x, c, s):
    """x [n, H, D], c / s [n, R / 2]."""
    R = case["rot"]
    c, s = c[:, None], s[:, None]
    if case["inter"]:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _views4(case, pool):
    """The (block, KV head, row) codes and scales of a 4-bit pool."""
    bs, D = case["bs"], case["D"]
    n = bs * D // 2
    return pool[..., :n].unflatten(-1, (bs, D // 2)), pool[..., n:n + bs * D // 32].unflatten(-1, (bs, D // 32))


def _put4(case, pool, slots, x):
    codes, scales = _views4(case, pool)
    b, o = slots // case["bs"], slots % case["bs"]
    x = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(x.abs().amax(-1))                 # amax = m 2^e, 1/2 <= m < 1
    e = torch.where(m < 0.875, e - 3, e - 2).clamp(-126, 127)
    y = torch.ldexp(x, -e[..., None])
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step                     # ties to even
    code = torch.where(a <= 2, 2 * a, torch.where(a < 6, a + 2, 7)).to(torch.uint8) + 8 * (y < 0).to(torch.uint8)
    code = code.flatten(-2)
    codes[b, :, o] = code[..., 0::2] + 16 * code[..., 1::2]
    scales[b, :, o] = (e + 127).to(torch.uint8)


_CODE = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _get4(case, pool, slots, f):
    """Rows [n, Hkv, D] of a 4-bit pool as the values they stand for."""
    codes, scales = _views4(case, pool)
    b, o = slots // case["bs"], slots % case["bs"]
    table = torch.tensor(_CODE + [-x for x in _CODE], dtype=f, device=pool.device)
    pair = torch.stack([table[:, None].expand(16, 16).t(), table[:, None].expand(16, 16)], -1).reshape(256, 2)
    x = pair[codes[b, :, o].to(torch.int32)].flatten(-2)           # low half first
    scale = torch.ldexp(torch.ones((), dtype=f, device=pool.device), scales[b, :, o].to(torch.int32) - 127)
    return (x.unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _attention(case, s, f):
    """softmax(q k^T / sqrt(D)) v over each row's visible keys, in the type f."""
    Hq, Hkv, D, bs, W, S = (case[x] for x in ("Hq", "Hkv", "D", "bs", "window", "sinks"))
    G, step = Hq // Hkv, 1024
    out = torch.empty(s["q"].shape, dtype=f, device="cuda")
    row = 0
    for i, (c, n) in enumerate(zip(s["ctx"], s["ql"])):
        for r0 in range(0, n, step):
            r1 = min(n, r0 + step)
            first, end = _first(case, c + r0), c + r1
            key = torch.arange(first, end, device="cuda")
            if first and S:
                key = torch.cat([torch.arange(min(S, first), device="cuda"), key])
            slot = s["bt"][i, key // bs].to(torch.int64) * bs + key % bs
            kv = [_get4(case, s[t], slot, f) if case["kv"] == "4" else s[t][slot].to(f) for t in ("k_cache", "v_cache")]
            p = c + torch.arange(r0, r1, device="cuda")[:, None]
            seen = key <= p
            if W:
                seen &= (key > p - W) | (key < S)
            q = s["q"][row + r0:row + r1].to(f)
            for h in range(Hkv):
                kh, vh = kv[0][:, h].contiguous(), kv[1][:, h].contiguous()
                sc = (q[:, h * G:(h + 1) * G].reshape(-1, D) @ kh.t().contiguous()) / math.sqrt(D)
                sc = sc.view(-1, G, kh.shape[0]).masked_fill(~seen[:, None], -math.inf)
                e = torch.exp(sc - sc.amax(-1, keepdim=True))
                o = (e.view(-1, kh.shape[0]) @ vh).view(-1, G, D) / e.sum(-1, keepdim=True)
                out[row + r0:row + r1, h * G:(h + 1) * G] = o
        row += n
    return out


# ------------------------------------------------------------------ work
def work(case):
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    e = SIZES[case["dtype"]]
    if case["kind"] != "attn":
        n = case["n"]
        kv = 2 * Hkv * (D // 32 * 17 if case["kind"] == "write4" else D * e)
        nbytes = n * ((2 * Hq + 2 * Hkv) * D * e + kv + 16)
        if case["kind"] == "write4":                       # read back: codes in, values out
            nbytes += n * (kv + 2 * Hkv * D * e + 8)
        return {"bytes": nbytes, "flops": 3 * n * (Hq + Hkv) * case["rot"]}
    ctx, ql = _lengths(case)
    W, S = case["window"], case["sinks"]
    keys = pairs = blocks = 0
    for c, n in zip(ctx, ql):
        p = np.arange(c, c + n, dtype=np.int64)
        pairs += int((np.minimum(p + 1, W) + np.minimum(S, np.maximum(0, p + 1 - W))).sum() if W else (p + 1).sum())
        used = c + n - max(0, _first(case, c) - S)
        keys += used
        blocks += -(-used // case["bs"])
    kv = 2 * Hkv * (D // 32 * 17 if case["kv"] == "4" else D * SIZES[case["kv"]])
    return {"bytes": keys * kv + 2 * sum(ql) * Hq * D * e + 4 * blocks, "flops": 4 * Hq * D * pairs}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    f = torch.float64
    if case["kind"] == "attn":
        return _exact_attention(case, _attn_inputs(case, seed))
    s = _rotary_inputs(case, seed)
    R, (freq, m) = case["rot"], _frequencies(case, f)
    z = torch.polar(torch.tensor(m, dtype=f).cuda(), s["pos"].to(f)[:, None, None] * freq.cuda())

    def turn(x):                                           # pairs as complex numbers
        x = x.to(f).clone()
        at = (slice(0, R, 2), slice(1, R, 2)) if case["inter"] else (slice(0, R // 2), slice(R // 2, R))
        y = torch.complex(x[..., at[0]], x[..., at[1]]) * z
        x[..., at[0]], x[..., at[1]] = y.real, y.imag
        return x

    q, k, v = turn(s["q"]), turn(s["k"]), s["v"].to(f)
    if case["kind"] == "write4":
        return q, _round4(k), _round4(v)
    kc, vc = s["k_cache"].to(f), s["v_cache"].to(f)
    kc[s["slots"]], vc[s["slots"]] = k, v
    return q, kc, vc


def _round4(x):
    """Each value as the nearest code of its block (ties to the even code)."""
    x = x.unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(top.clamp_min(1e-300))) - 2)
    scale = torch.where(top >= 7 * scale, 2 * scale, scale)
    scale = torch.where(top >= 7 * scale, 2 * scale, scale).clamp_min(2.0 ** -126)
    a = (x / scale).abs()
    y = 0.5 * ((a > 0.25).to(x) + (a >= 0.75) + (a > 1.25) + (a >= 1.75)) + (a > 2.5).to(x) + (a >= 3.5) + 2.0 * (a > 5)
    return (torch.where(x < 0, -y, y) * scale).flatten(-2)


def _exact_attention(case, s):
    Hkv, D, bs, W, S = (case[x] for x in ("Hkv", "D", "bs", "window", "sinks"))
    G, f = case["Hq"] // Hkv, torch.float64
    code = torch.tensor(_CODE + [-x for x in _CODE], dtype=f, device="cuda")

    def rows(pool, blk, off):
        if case["kv"] != "4":
            return pool[blk * bs + off].to(f)
        flat = pool.reshape(pool.shape[0], Hkv, -1)[blk]                       # [keys, Hkv, record]
        at = off[:, None, None] * (D // 2) + torch.arange(D // 2, device="cuda")
        b = torch.gather(flat, 2, at.expand(-1, Hkv, -1)).to(torch.int32)
        at = bs * D // 2 + off[:, None, None] * (D // 32) + torch.arange(D // 32, device="cuda")
        e = torch.gather(flat, 2, at.expand(-1, Hkv, -1)).to(f) - 127
        x = torch.empty(len(blk), Hkv, D, dtype=f, device="cuda")
        x[..., 0::2], x[..., 1::2] = code[b % 16], code[b // 16]
        return x * torch.exp2(e).repeat_interleave(32, -1)

    out, row = torch.empty(s["q"].shape, dtype=f, device="cuda"), 0
    for i, (c, n) in enumerate(zip(s["ctx"], s["ql"])):
        for r0 in range(0, n, 512):
            m = min(512, n - r0)
            pos = torch.arange(c + r0, c + r0 + m, device="cuda")
            key = torch.arange(c + r0 + m, device="cuda")
            if W:
                key = key[(key > c + r0 - W) | (key < S)]
            hidden = key[None, :] > pos[:, None]
            if W:
                hidden |= (key[None, :] <= pos[:, None] - W) & (key[None, :] >= S)
            blk, off = s["bt"][i][key // bs].to(torch.int64), key % bs
            # long contexts: a block of keys at a time would only reorder the sums
            k, v = rows(s["k_cache"], blk, off), rows(s["v_cache"], blk, off)
            q = s["q"][row + r0:row + r0 + m].to(f).view(m, Hkv, G, D)
            for h in range(Hkv):
                sc = q[:, h].reshape(m * G, D).mm(k[:, h].t().contiguous()).view(m, G, -1) / math.sqrt(D)
                p = torch.softmax(sc.masked_fill(hidden[:, None], -math.inf), -1)
                out[row + r0:row + r0 + m].view(m, Hkv, G, D)[:, h] = p.view(m * G, -1).mm(v[:, h].contiguous()).view(m, G, D)
        row += n
    return out
