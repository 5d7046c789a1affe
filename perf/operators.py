"""The serving step's operators around the paged cache, as they are timed.

Three operators of one layer of a decode or prefill step:

* ``norm_rope``: the RMS norm of every query and key head and the rotation by
  the token's position, in one pass over the projection's output;
* ``write_rope``: the same on the way into the paged cache, with the values
  stored and the queries returned by the same call;
* ``shared``: paged decode attention of a batch whose sequences begin with the
  same prompt in the same pages, that prompt attended once for all of them.

Sizes are those of this repository's benchmark configurations and tests, or
between them.  Lengths and positions come from the case alone
(``length_seed``), so that the work and the shapes of a case are known; values
and page orders come from ``prepare``'s seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "e4m3": 1, "f32": 4}
FP8_MAX = 448.0

# (query heads, KV heads, head_dim): the benchmark's and the tests' head shapes
HEADS = [(32, 8, 128), (64, 8, 128), (16, 8, 128), (8, 8, 128), (40, 8, 128), (32, 4, 128), (64, 4, 128),
         (32, 1, 128), (64, 8, 64), (32, 8, 64), (32, 8, 256), (16, 8, 256)]


def _rope(op, tokens, seqs, heads, dtype, *, norm, rotary, interleaved=False, table="f32", kv=None, length_seed=1,
          name=None):
    hq, hkv, d = heads
    c = dict(op=op, tokens=tokens, seqs=seqs, q_heads=hq, kv_heads=hkv, head_dim=d, dtype=dtype, norm=norm,
             rotary=rotary, interleaved=interleaved, table=table, kv=kv or dtype, length_seed=length_seed)
    if name:
        c["name"] = name
    return c


def _shared(batch, heads, kv, prefix, lo, hi, *, sinks="none", short=0, length_seed=1, name=None):
    hq, hkv, d = heads
    c = dict(op="shared", batch=batch, q_heads=hq, kv_heads=hkv, head_dim=d, kv=kv, prefix=prefix, lo=lo, hi=hi,
             sinks=sinks, short=short, length_seed=length_seed)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # One token of one conversation: nothing but latency and launches.
        _rope("norm_rope", 1, 1, (32, 8, 128), "bf16", norm=True, rotary=128, name="norm_rope_one"),
        # The prompts of a prefill batch, sequence after sequence.
        _rope("norm_rope", 16384, 5, (32, 8, 128), "bf16", norm=True, rotary=128, length_seed=2,
              name="norm_rope_prefill"),
        # Neighbouring pairs, half of the head rotated, 16-bit tables, an odd number of tokens.
        _rope("norm_rope", 1237, 3, (64, 8, 64), "f16", norm=False, rotary=32, interleaved=True, table="f16",
              length_seed=3, name="norm_rope_partial"),
        # One new token for each of 32 sequences into pools of their type.
        _rope("write_rope", 32, 32, (32, 8, 128), "bf16", norm=True, rotary=128, length_seed=4,
              name="write_rope_step"),
        # One token of one conversation, no norms.
        _rope("write_rope", 1, 1, (32, 8, 128), "f16", norm=False, rotary=128, length_seed=5, name="write_rope_one"),
        # A long prefill quantised into scattered e4m3 pages.
        _rope("write_rope", 28001, 8, (32, 8, 128), "bf16", norm=True, rotary=128, kv="e4m3", length_seed=6,
              name="write_rope_prefill_e4m3"),
        # Four samples of one short prompt, a few tokens in.
        _shared(4, (32, 8, 128), "f16", 1024, 1, 100, length_seed=7, name="shared_small"),
        # A server whose system prompt is shared by 32 conversations.
        _shared(32, (32, 8, 128), "bf16", 8192, 16, 1024, length_seed=8, name="shared_server"),
        # A long document in an e4m3 cache, 64 questions about it, sink logits.
        _shared(64, (32, 8, 128), "e4m3", 32768, 16, 512, sinks="exp", length_seed=9, name="shared_document_e4m3"),
        # head_dim 64, eight query heads per KV head, a prompt that ends inside a page, some rows shorter than it.
        _shared(17, (64, 8, 64), "f16", 2109, 1, 300, sinks="exp", short=3, length_seed=10, name="shared_d64_ragged"),
        # head_dim 256, few sequences with long turns of their own.
        _shared(6, (32, 8, 256), "bf16", 4096, 500, 4000, length_seed=11, name="shared_d256"),
        # Many samples of one prompt (the widest batch).
        _shared(256, (32, 8, 128), "f16", 4096, 1, 256, length_seed=12, name="shared_many_samples"),
    ]


def draw(rng: random.Random):
    """A case of the same ranges: any operator, sizes spread over their logarithms."""
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    heads = rng.choice(HEADS)
    op = rng.choice(["norm_rope", "write_rope", "shared", "shared"])
    seed = rng.randrange(1 << 30)
    # the same bytes per token as the listed head shape allow the same number of tokens
    weight = max((heads[0] + 2 * heads[1]) * heads[2] / (48 * 128), 1.0)
    if op != "shared":
        tokens = log_int(1, int(28000 / weight))
        rotary = rng.choice([heads[2], heads[2], heads[2] // 2, 32])
        dtype = rng.choice(["f16", "bf16", "bf16", "f32"])
        kv = None
        if op == "write_rope":
            kv = rng.choice(["f16", "bf16", "e4m3"]) if dtype == "f32" else rng.choice([dtype, "e4m3"])
        if dtype == "f32":
            tokens = max(1, tokens // 2)
        return _rope(op, tokens, min(tokens, log_int(1, 64)), heads, dtype, norm=rng.random() < 0.5, rotary=rotary,
                     interleaved=rng.random() < 0.3, table=rng.choice(["f32", "f32", "bf16"]), kv=kv,
                     length_seed=seed)
    batch = log_int(1, 256)
    most = 2_100_000 * 32 * 128 / max(heads[0] * heads[2], 32 * 128)  # batch x prefix of the largest listed case
    prefix = log_int(64, int(max(65, min(32768, most / batch))))
    hi = log_int(1, int(max(2, min(4096, 32768 * 8 * 128 / max(heads[1] * heads[2], 1024) / batch))))
    sinks = rng.choice(["none", "linear", "exp", "exp"])
    short = min(batch - 1, rng.choice([0, 0, 1, 3])) if sinks == "exp" else 0
    return _shared(batch, heads, rng.choice(["f16", "bf16", "e4m3"]), prefix, rng.randint(1, hi), hi, sinks=sinks,
                   short=short, length_seed=seed)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _token_lens(c):
    """Tokens of each sequence of a rope case (they add up to the case's), and of its cache before them."""
    r = random.Random(c["length_seed"])
    cuts = sorted(r.sample(range(1, c["tokens"]), c["seqs"] - 1)) if c["seqs"] > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [c["tokens"]])], [r.randrange(4000) for _ in range(c["seqs"])]


def _seq_lens(c):
    """Whole lengths of a shared case's sequences; the last ``short`` of them end inside the prefix, the very last
    one empty (a padded batch slot)."""
    r = random.Random(c["length_seed"])
    lens = [c["prefix"] + r.randint(c["lo"], c["hi"]) for _ in range(c["batch"])]
    for i in range(c["short"]):
        lens[-1 - i] = r.randint(1, c["prefix"]) if i else 0
    return lens


def _pages(c):
    """Pages that all sequences share, and each sequence's own."""
    common = c["prefix"] // PAGE
    return common, [max(0, -(-n // PAGE) - common) for n in _seq_lens(c)]


def _quantize(x):
    scale = x.abs().max().clamp(min=1e-12) / FP8_MAX
    return (x / scale).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn), scale


def _prepare_rope(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    n, hq, hkv, d = c["tokens"], c["q_heads"], c["kv_heads"], c["head_dim"]
    dt = DT[c["dtype"]]
    s = dict(case=c)
    # the projection's output: queries, keys and values of a token side by side
    width = (hq + 2 * hkv) * d
    s["qkv"] = torch.randn(n, width, generator=g, device=dev).to(dt)
    s["q"] = s["qkv"][:, :hq * d].view(n, hq, d)
    s["k"] = s["qkv"][:, hq * d:(hq + hkv) * d].view(n, hkv, d)
    s["v"] = s["qkv"][:, (hq + hkv) * d:].view(n, hkv, d)
    s["qw"] = s["kw"] = None
    if c["norm"]:
        s["qw"] = (1 + 0.2 * torch.randn(d, generator=g, device=dev)).to(dt)
        s["kw"] = (1 + 0.2 * torch.randn(d, generator=g, device=dev)).to(dt)
    # every sequence's tokens follow what its cache holds
    lens, past = (torch.tensor(t, device=dev) for t in _token_lens(c))
    at = torch.cat([torch.arange(m, device=dev) for m in lens.tolist()])
    seq = torch.repeat_interleave(torch.arange(len(lens), device=dev), lens)
    s["positions"] = past[seq] + at
    rows = 4000 + c["tokens"]
    half = c["rotary"] // 2
    freq = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
    angle = torch.arange(rows, dtype=torch.float64, device=dev)[:, None] * freq
    s["cos"], s["sin"] = angle.cos().to(DT[c["table"]]), angle.sin().to(DT[c["table"]])
    if c["op"] == "write_rope":
        # scattered pages, as a fragmented pool gives them: the tokens of a sequence fill pages in order
        first = past % PAGE
        pages = -(-(first + lens) // PAGE)
        base = torch.cumsum(pages, 0) - pages
        total = int(pages.sum())
        P = total + total // 10 + 1
        perm = torch.randperm(P, generator=g, device=dev)
        row = first[seq] + at
        s["slots"] = perm[base[seq] + row // PAGE] * PAGE + row % PAGE
        e4m3 = c["kv"] == "e4m3"
        shape = (P, hkv, PAGE, d)
        s["k_pool"] = torch.zeros(shape, dtype=torch.uint8 if e4m3 else DT[c["kv"]], device=dev).view(DT[c["kv"]])
        s["v_pool"] = torch.zeros_like(s["k_pool"])
        s["k_scale"] = torch.tensor(0.013, device=dev) if e4m3 else None
        s["v_scale"] = torch.tensor(0.011, device=dev) if e4m3 else None
    return s


def _prepare_shared(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    B, hq, hkv, d, kv = c["batch"], c["q_heads"], c["kv_heads"], c["head_dim"], c["kv"]
    lens = _seq_lens(c)
    common, rest = _pages(c)
    P = common + sum(rest)
    P += P // 10 + 1
    perm = torch.randperm(P, generator=g, device=dev).to(torch.int32).cpu()
    table = torch.full((B, common + max(max(rest), 1)), -1, dtype=torch.int32)
    table[:, :common] = perm[:common]
    off = common
    for b, m in enumerate(rest):
        table[b, common:common + m] = perm[off:off + m]
        off += m
    s = dict(case=c, table=table.to(dev), lens=torch.tensor(lens, dtype=torch.int32, device=dev), common=common)
    qdt = DT["bf16" if kv == "e4m3" else kv]
    s["q"] = torch.randn(B, hq, d, generator=g, device=dev).to(qdt)
    s["k_scale"] = s["v_scale"] = None
    for name in ("k", "v"):
        x = torch.randn(P, hkv, PAGE, d, generator=g, device=dev)
        if kv == "e4m3":
            s[name], s[name + "_scale"] = _quantize(x)
        else:
            s[name] = x.to(DT[kv])
    s["sinks"] = None
    if c["sinks"] != "none":
        s["sinks"] = torch.randn(hq, generator=g, device=dev) * (0.1 if c["sinks"] == "linear" else 1.0)
    return s


def prepare(case, seed):
    s = _prepare_shared(case, seed) if case["op"] == "shared" else _prepare_rope(case, seed)
    if own:
        from fskernels import hip
        s["hip"] = hip
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if c["op"] == "norm_rope":
        return _run_norm_rope(s, c)
    if c["op"] == "write_rope":
        return _run_write_rope(s, c)
    return _run_shared(s, c)


def _norm_rotate(x, weight, cos, sin, interleaved):
    """x [n, H, D] with cos and sin [n, R / 2], in fp32."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    half = cos.shape[-1]
    cos, sin = cos.float()[:, None], sin.float()[:, None]
    y = x.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def _run_norm_rope(s, c):
    if own:
        return s["hip"].qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["positions"], q_weight=s["qw"],
                                     k_weight=s["kw"], eps=1e-6, interleaved=c["interleaved"])
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    return (_norm_rotate(s["q"], s["qw"], cos, sin, c["interleaved"]).to(s["q"].dtype),
            _norm_rotate(s["k"], s["kw"], cos, sin, c["interleaved"]).to(s["k"].dtype))


def _run_write_rope(s, c):
    if own:
        q = s["hip"].paged_kv_write_rope(s["q"], s["k"], s["v"], s["k_pool"], s["v_pool"], s["slots"], s["cos"],
                                         s["sin"], s["positions"], q_weight=s["qw"], k_weight=s["kw"], eps=1e-6,
                                         interleaved=c["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return q, s["k_pool"], s["v_pool"]
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    q = _norm_rotate(s["q"], s["qw"], cos, sin, c["interleaved"]).to(s["q"].dtype)
    k = _norm_rotate(s["k"], s["kw"], cos, sin, c["interleaved"])
    page, row = s["slots"] // PAGE, s["slots"] % PAGE
    for pool, x, scale in ((s["k_pool"], k, s["k_scale"]), (s["v_pool"], s["v"].float(), s["v_scale"])):
        if scale is not None:
            x = (x / scale).clamp(-FP8_MAX, FP8_MAX).to(pool.dtype)
            pool.view(torch.uint8)[page, :, row] = x.view(torch.uint8)
        else:
            pool[page, :, row] = x.to(pool.dtype)
    return q, s["k_pool"], s["v_pool"]


def _run_shared(s, c):
    if own:
        return s["hip"].paged_flash_decode_shared(s["q"], s["k"], s["v"], s["table"], s["lens"], PAGE, c["prefix"],
                                                  s_aux=s["sinks"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                                  sink_mode="linear" if c["sinks"] == "linear" else "exp")
    B, hq, hkv, d, common = c["batch"], c["q_heads"], c["kv_heads"], c["head_dim"], s["common"]
    G = hq // hkv
    q = s["q"].float().view(B, hkv, G, d)
    table = s["table"].long().clamp(min=0)

    def pages(pool, scale, ids):
        x = pool.view(torch.uint8)[ids].view(pool.dtype) if pool.element_size() == 1 else pool[ids]
        x = x.float()
        return x if scale is None else x * scale

    # the common pages once: [hkv, T, d]
    kp, vp = (pages(s[n], s[n + "_scale"], table[0, :common]).transpose(0, 1).reshape(hkv, -1, d) for n in "kv")
    rows = q.transpose(0, 1).reshape(hkv, B * G, d)
    sp = torch.matmul(rows, kp.transpose(1, 2).contiguous()).view(hkv, B, G, -1).transpose(0, 1)
    # each sequence's own pages: [B, hkv, S, d]
    ko, vo = (pages(s[n], s[n + "_scale"], table[:, common:]).transpose(1, 2).reshape(B, hkv, -1, d) for n in "kv")
    so = torch.matmul(q, ko.transpose(2, 3).contiguous())
    x = torch.cat([sp, so], -1) * d ** -0.5
    inside = torch.arange(x.shape[-1], device=x.device) < s["lens"][:, None]
    x = x.masked_fill(~inside[:, None, None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    z = None if s["sinks"] is None else s["sinks"].view(1, hkv, G, 1)
    if c["sinks"] == "exp":
        m = torch.maximum(m, z)
    p = torch.exp(x - m)
    den = p.sum(-1, keepdim=True)
    if z is not None:
        den = den + (torch.exp(z - m) if c["sinks"] == "exp" else z)
    n = sp.shape[-1]
    pp = p[..., :n].transpose(0, 1).reshape(hkv, B * G, n)
    out = torch.matmul(pp, vp).view(hkv, B, G, d).transpose(0, 1) + torch.matmul(p[..., n:].contiguous(), vo)
    return (out / den).reshape(B, hq, d).to(s["q"].dtype)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    hq, hkv, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    if c["op"] == "shared":
        lens = _seq_lens(c)
        longest = min(max(lens), c["prefix"])
        tokens = longest + sum(max(0, n - c["prefix"]) for n in lens)
        nbytes = tokens * hkv * d * 2 * SIZE[c["kv"]] + 2 * c["batch"] * hq * d * 2 + 4 * c["batch"]
        nbytes += 4 * (-(-longest // PAGE) + sum(_pages(c)[1]))
        return {"bytes": nbytes, "flops": 4 * d * hq * sum(lens)}
    n, e, half = c["tokens"], SIZE[c["dtype"]], c["rotary"] // 2
    table = min(n, 4000 + n) * half * 2 * SIZE[c["table"]]
    flops = n * (hq + hkv) * (3 * c["rotary"] + (4 * d if c["norm"] else 0))
    if c["op"] == "norm_rope":
        return {"bytes": 2 * n * (hq + hkv) * d * e + table + 8 * n, "flops": flops}
    nbytes = n * (hq + 2 * hkv) * d * e + n * hq * d * e + 2 * n * hkv * d * SIZE[c["kv"]] + table + 16 * n
    return {"bytes": nbytes, "flops": flops}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_rotated(x, weight, cos, sin, interleaved):
    """Each pair as a complex number times cos + i sin."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * weight.double()
    r = 2 * cos.shape[-1]
    turn = torch.complex(cos.double(), sin.double())[:, None]
    pairs = x[..., :r].unflatten(-1, (-1, 2)) if interleaved else x[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    head = z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)
    return torch.cat([head, x[..., r:]], -1)


def exact(case, seed):
    c = case
    if c["op"] == "shared":
        s = _prepare_shared(c, seed)
        hkv, d = c["kv_heads"], c["head_dim"]
        out = torch.zeros(c["batch"], c["q_heads"], d, dtype=torch.float64, device=s["q"].device)
        fp8 = c["kv"] == "e4m3"
        kv = [s[n].float() if fp8 else s[n] for n in "kv"]
        scales = [s[n].double() if fp8 else 1.0 for n in ("k_scale", "v_scale")]
        for b, n in enumerate(_seq_lens(c)):
            if n == 0:
                continue  # nothing to attend: only the sink, whose value is zero
            ids = s["table"][b, :-(-n // PAGE)].long()
            k, v = (t[ids].transpose(0, 1).reshape(hkv, -1, d)[:, :n].double() * sc for t, sc in zip(kv, scales))
            q = s["q"][b].double().view(hkv, -1, d)
            x = torch.matmul(q, k.transpose(1, 2).contiguous()) / math.sqrt(d)
            top = x.amax(-1, keepdim=True)
            w = torch.exp(x - top)
            total = w.sum(-1, keepdim=True)
            if s["sinks"] is not None:
                z = s["sinks"].double().view(hkv, -1, 1)
                total = total + (z if c["sinks"] == "linear" else torch.exp(z - top))
            out[b] = (torch.matmul(w, v) / total).view(-1, d)
        return out
    s = _prepare_rope(c, seed)
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    q = _exact_rotated(s["q"], s["qw"], cos, sin, c["interleaved"])
    k = _exact_rotated(s["k"], s["kw"], cos, sin, c["interleaved"])
    if c["op"] == "norm_rope":
        return q, k
    pools = []
    for pool, x, scale in ((s["k_pool"], k, s["k_scale"]), (s["v_pool"], s["v"].double(), s["v_scale"])):
        full = pool.float().double()
        if scale is not None:
            x = (x / scale.double()).clamp(-FP8_MAX, FP8_MAX)
        full[s["slots"] // PAGE, :, s["slots"] % PAGE] = x
        pools.append(full)
    return (q, *pools)
