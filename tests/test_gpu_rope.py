"""GPU parity of the norm-and-rotation operators (qk_norm_rope,
paged_kv_write_rope) against their formula in float64.

Bars, derived: the kernels compute in fp32 and round once.  A value a c - b s
carries at most 18 fp32 roundings relative to |a c| + |b s| (the norm's sum of
squares is at most 16 multiply-adds and 4 adds per lane and row, plus the mean's:
21 of its roundings, halved by the root; root, quotient, two products and the
rotation's two: 17), then half a step of the stored type.  Value rows are the
KV write's, bit for bit.
"""
import ctypes

import pytest
import torch

from fasterkernels_amd import native as nat
from fskernels.hip import paged_kv_write, paged_kv_write_rope, qk_norm_rope

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
# half of the smallest step (subnormals)
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134, "f32": 2.0 ** -150, "e4m3": 2.0 ** -10}


def oracle(x, w, cos, sin, row, eps, interleaved):
    """(value, |a c| + |b s|) of every element in float64, on the host."""
    x = x.detach().cpu().double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.cpu().double()
    if cos is None:
        return x, x.abs()
    c, s = (t.cpu().double()[row.cpu()][:, None] for t in (cos, sin))
    half = c.shape[-1]
    y, m = x.clone(), x.abs()
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    m[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    m[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, m


def close(got, want, mag, dt, what):
    step = torch.finfo(DT[dt]).eps / 2
    tol = mag * (18 * 2.0 ** -24) + step * want.abs() * (1 + 2.0 ** -10) + TINY[dt]
    err = (got.cpu().float().double() - want).abs()
    assert (err <= tol).all(), f"{what}: worst {(err / tol).max().item():.3f} of the bar"


def table(rows, half, dt, seed):
    g = torch.Generator().manual_seed(seed)
    angle = torch.rand(rows, half, generator=g, dtype=torch.float64) * 6.283
    return angle.cos().to(DT[dt]).to(DEV), angle.sin().to(DT[dt]).to(DEV)


def projection(n, hq, hkv, d, dt, seed, pad=0):
    """q, k and v as views of one projection's output (``pad`` elements between tokens)."""
    g = torch.Generator().manual_seed(seed)
    width = (hq + 2 * hkv) * d
    x = torch.randn(n, width + pad, generator=g).to(DT[dt]).to(DEV)[:, :width]
    q, k, v = x.split([hq * d, hkv * d, hkv * d], dim=1)
    return (q.unflatten(1, (hq, d)), k.unflatten(1, (hkv, d)), v.unflatten(1, (hkv, d)))


def weights(d, dt, seed):
    g = torch.Generator().manual_seed(seed)
    return [(1 + 0.3 * torch.randn(d, generator=g)).to(DT[dt]).to(DEV) for _ in range(2)]


CASES = [
    # n, hq, hkv, d, dtype, rotary, interleaved, norm, table dtype
    (1, 32, 8, 128, "bf16", 128, False, True, "f32"),
    (3, 32, 8, 128, "f16", 128, True, True, "f16"),
    (37, 64, 8, 64, "f16", 32, True, False, "bf16"),
    (37, 16, 8, 256, "bf16", 64, False, True, "f32"),
    (5, 5, 1, 80, "f32", 80, False, True, "f32"),
    (5, 3, 3, 96, "bf16", 48, True, True, "f32"),
    (7, 2, 1, 16, "f32", 16, True, True, "f32"),
    (7, 9, 3, 192, "f16", 192, False, True, "f32"),
    (2, 1, 1, 32, "f32", 16, False, False, "f32"),
    (1200, 32, 8, 128, "bf16", 128, False, True, "bf16"),
    (1200, 20, 4, 64, "f32", 64, True, True, "f32"),
]


@pytest.mark.parametrize("n,hq,hkv,d,dt,rotary,inter,norm,tdt", CASES)
def test_norm_rope(n, hq, hkv, d, dt, rotary, inter, norm, tdt):
    q, k, _ = projection(n, hq, hkv, d, dt, n + d, pad=16)
    cos, sin = table(97, rotary // 2, tdt, 1)
    pos = torch.randint(0, 97, (n,), generator=torch.Generator().manual_seed(2)).to(DEV)
    qw, kw = weights(d, dt, 3) if norm else (None, None)
    qo, ko = qk_norm_rope(q, k, cos, sin, pos, q_weight=qw, k_weight=kw, eps=1e-6, interleaved=inter)
    assert qo.shape == (n, hq, d) and ko.shape == (n, hkv, d) and qo.dtype is DT[dt] and qo.is_contiguous()
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        close(got, *oracle(x, w, cos, sin, pos, 1e-6, inter), dt, "rotated rows")


def test_tables_without_positions_repeat():
    q, k, _ = projection(12, 4, 2, 64, "f32", 5)
    cos, sin = table(4, 32, "f32", 6)
    row = torch.arange(12) % 4
    qo, ko = qk_norm_rope(q, k, cos, sin)
    close(qo, *oracle(q, None, cos, sin, row, 0, False), "f32", "four rows for twelve tokens")
    # tables with a row stride of their own (the halves of a doubled table)
    wide_c, wide_s = torch.cat([cos, cos], 1), torch.cat([sin, sin], 1)
    again = qk_norm_rope(q, k, wide_c[:, :32], wide_s[:, :32])
    assert torch.equal(again[0], qo) and torch.equal(again[1], ko)


def test_positions_outside_the_table_take_its_ends():
    q, k, _ = projection(5, 4, 2, 64, "f16", 7)
    cos, sin = table(10, 32, "f32", 8)
    pos = torch.tensor([-1, -(1 << 60), 9, 10, 1 << 60], device=DEV)
    got = qk_norm_rope(q, k, cos, sin, pos)
    want = qk_norm_rope(q, k, cos, sin, torch.tensor([0, 0, 9, 9, 9], device=DEV))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    small = qk_norm_rope(q, k, cos, sin, torch.tensor([0, 0, 9, 9, 9], dtype=torch.int32, device=DEV))
    assert torch.equal(small[0], want[0])


def test_norms_alone_and_one_weight():
    q, k, _ = projection(9, 8, 2, 128, "bf16", 9)
    qw, kw = weights(128, "f32", 10)
    qo, ko = qk_norm_rope(q, k, None, None, q_weight=qw, k_weight=kw, eps=1e-5)
    close(qo, *oracle(q, qw, None, None, None, 1e-5, False), "bf16", "q norm")
    close(ko, *oracle(k, kw, None, None, None, 1e-5, False), "bf16", "k norm")
    qo, ko = qk_norm_rope(q, k, None, None, k_weight=kw)
    assert torch.equal(qo, q) and not torch.equal(ko, k)


def test_rows_keep_to_themselves():
    """An infinity, a NaN and a row of zeros change their own row only; a row of
    zeros normalises to zeros."""
    q, k, _ = projection(6, 4, 2, 128, "f16", 11)
    cos, sin = table(6, 64, "f32", 12)
    qw, kw = weights(128, "f16", 13)
    base = qk_norm_rope(q, k, cos, sin, q_weight=qw, k_weight=kw)
    q2 = q.clone()
    q2[1, 2, 5], q2[3, 0, 100], q2[4, 1] = float("inf"), float("nan"), 0
    qo, ko = qk_norm_rope(q2, k, cos, sin, q_weight=qw, k_weight=kw)
    same = torch.ones(6, 4, dtype=torch.bool)
    same[1, 2] = same[3, 0] = same[4, 1] = False
    assert torch.equal(qo[same.to(DEV)], base[0][same.to(DEV)]) and torch.equal(ko, base[1])
    assert qo[3, 0].isnan().all() and (qo[4, 1] == 0).all()
    assert qo[1, 2, 5].isnan()  # inf / inf, as the formula gives


@pytest.mark.parametrize("n", [0, 4])
def test_odd_tensors(n):
    """No tokens; rows at an odd address, with gaps, expanded or lazily negated."""
    q, k, _ = projection(n, 4, 2, 64, "f16", 14)
    cos, sin = table(max(n, 1), 32, "f32", 15)
    want = qk_norm_rope(q, k, cos, sin, torch.arange(n, device=DEV))
    if n == 0:
        assert want[0].shape == (0, 4, 64)
        return
    flat = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape).copy_(q)
    gaps = torch.empty(n, 4, 64, 2, dtype=q.dtype, device=DEV)[..., 0].copy_(q)
    for x in (flat, gaps, q.neg().clone()._neg_view()):
        got = qk_norm_rope(x, k, cos, sin, torch.arange(n, device=DEV))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = q[:1].expand(n, 4, 64)
    got = qk_norm_rope(one, k, cos, sin)[0]
    assert torch.equal(got, qk_norm_rope(one.contiguous(), k, cos, sin)[0])


def test_outputs_in_place_through_the_c_abi():
    n, hq, hkv, d = 130, 8, 2, 128
    q, k, _ = projection(n, hq, hkv, d, "bf16", 16)
    cos, sin = table(n, 64, "f32", 17)
    qw, kw = weights(d, "bf16", 18)
    want = qk_norm_rope(q, k, cos, sin, q_weight=qw, k_weight=kw)
    nat.check(nat.load().fsk_qk_norm_rope(
        q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), n, cos.data_ptr(),
        cos.stride(0), sin.data_ptr(), sin.stride(0), n, nat.FSK_F32, d, 0, None, qw.data_ptr(), kw.data_ptr(),
        nat.FSK_BF16, ctypes.c_float(1e-6), q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0),
        k.stride(1), hq, hkv, d, nat.FSK_BF16, nat.stream_handle(0)))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


# ---------------------------------------------------------------------------
# into the paged cache
# ---------------------------------------------------------------------------
def pools(P, hkv, d, dt, page=16):
    fill = {"f16": 0x5A5A, "bf16": 0x5A5A, "e4m3": 0x5A}[dt]
    raw = torch.uint8 if dt == "e4m3" else torch.int16
    return [torch.full((P, hkv, page, d), fill, dtype=raw, device=DEV).view(DT[dt]) for _ in range(2)]


def raw(t):
    return t.view(torch.uint8 if t.element_size() == 1 else torch.int16)


WRITES = [
    # n, hq, hkv, d, source, pool, scaled, rotary, interleaved, norm, page size
    (1, 32, 8, 128, "f16", "f16", False, 128, False, False, 16),
    (33, 32, 8, 128, "bf16", "bf16", False, 128, False, True, 16),
    (33, 32, 8, 128, "bf16", "e4m3", True, 128, False, True, 16),
    (21, 8, 8, 64, "f16", "e4m3", False, 32, True, True, 32),
    (21, 7, 1, 256, "f32", "bf16", False, 256, False, True, 16),
    (21, 5, 5, 80, "f32", "f16", False, 16, True, False, 4),
    (900, 0, 8, 128, "bf16", "e4m3", True, 128, False, False, 16),
    (900, 64, 4, 64, "f32", "e4m3", True, 64, False, True, 16),
]


@pytest.mark.parametrize("n,hq,hkv,d,src,pool,scaled,rotary,inter,norm,page", WRITES)
def test_write_rope(n, hq, hkv, d, src, pool, scaled, rotary, inter, norm, page):
    q, k, v = projection(n, max(hq, 1), hkv, d, src, n + d + 1)
    q = q if hq else None
    P = n // page + 9
    g = torch.Generator().manual_seed(20)
    slots = torch.randperm(P * page, generator=g)[:n]
    if n > 3:
        slots[1], slots[3] = -1, P * page  # skipped
    cos, sin = table(50, rotary // 2, "f32", 21)
    pos = torch.randint(0, 50, (n,), generator=g).to(DEV)
    qw, kw = weights(d, src, 22) if norm else (None, None)
    if not hq:
        qw = None
    ks, vs = (torch.tensor(0.017, device=DEV), torch.tensor(0.021, device=DEV)) if scaled else (None, None)
    kp, vp = pools(P, hkv, d, pool, page)
    k2, v2 = pools(P, hkv, d, pool, page)
    qo = paged_kv_write_rope(q, k, v, kp, vp, slots.to(DEV), cos, sin, pos, q_weight=qw, k_weight=kw, eps=1e-6,
                             interleaved=inter, k_scale=ks, v_scale=vs)
    if hq:
        close(qo, *oracle(q, qw, cos, sin, pos, 1e-6, inter), src, "queries")
    else:
        assert qo is None
    # values, and every row that is not written, as the KV write leaves them
    paged_kv_write(k, v, k2, v2, slots.to(DEV), k_scale=ks, v_scale=vs)
    assert torch.equal(raw(vp), raw(v2))
    ok = (slots >= 0) & (slots < P * page)
    touched = torch.zeros(P, page, dtype=torch.bool)
    touched[slots[ok] // page, slots[ok] % page] = True
    at = touched[:, None, :].expand(P, hkv, page).to(DEV)
    assert torch.equal(raw(kp)[~at], raw(pools(P, hkv, d, pool, page)[0])[~at])
    want, mag = oracle(k, kw, cos, sin, pos, 1e-6, inter)
    if scaled:
        want, mag = (want / ks.item()).clamp(-448, 448), mag / ks.item()
    got = kp.float()[slots[ok] // page, :, slots[ok] % page]
    close(got, want[ok], mag[ok], pool, "stored keys")


def test_write_without_norm_or_rotation_is_the_kv_write():
    n, hkv, d = 40, 4, 128
    _, k, v = projection(n, 1, hkv, d, "bf16", 23)
    k, v = k.clone(), v.clone()
    raw(v)[3, 1, 7], raw(v)[5, 0, 0] = 0x7F81, -0x0041  # NaN payloads are copied
    slots = torch.arange(n, device=DEV)
    a, b = pools(3, hkv, d, "bf16"), pools(3, hkv, d, "bf16")
    assert paged_kv_write_rope(None, k, v, *a, slots, None, None) is None
    paged_kv_write(k, v, *b, slots)
    assert torch.equal(raw(a[0]), raw(b[0])) and torch.equal(raw(a[1]), raw(b[1]))


def test_write_block_table_updates_and_non_finite_codes():
    n, hkv, d = 3, 2, 64
    _, k, v = projection(n, 1, hkv, d, "f32", 24)
    k = k.clone()
    k[0, 0, 3], k[1, 1, 5], k[2, 0, 9] = float("nan"), float("inf"), -1e30
    kp, vp = pools(2, hkv, d, "e4m3")
    k2, v2 = pools(2, hkv, d, "e4m3")
    one = torch.tensor(1.0, device=DEV)
    bt = torch.full((2, 300), -1, dtype=torch.int32, device=DEV)
    upd = torch.tensor([[i, i + 5] for i in range(290)] + [[600, 1], [-1, 1]], device=DEV)
    slots = torch.tensor([0, 17, 31], device=DEV)
    paged_kv_write_rope(None, k, v, kp, vp, slots, None, None, k_scale=one, v_scale=one, block_table=bt,
                        bt_updates=upd)
    paged_kv_write(k, v, k2, v2, slots, k_scale=one, v_scale=one)
    assert torch.equal(raw(kp), raw(k2)) and torch.equal(raw(vp), raw(v2))
    assert bt.view(-1)[:290].tolist() == [i + 5 for i in range(290)] and (bt.view(-1)[290:] == -1).all()
    # updates alone
    bt.fill_(-1)
    empty = k[:0]
    paged_kv_write_rope(None, empty, empty, kp, vp, slots[:0], None, None, k_scale=one, v_scale=one, block_table=bt,
                        bt_updates=upd)
    assert bt.view(-1)[:290].tolist() == [i + 5 for i in range(290)]


def test_graph_and_streams():
    """Captured once, replayed over changing inputs with eager calls between; and
    on a stream of its own."""
    n, hq, hkv, d = 16, 32, 8, 128
    q, k, v = [t.contiguous() for t in projection(n, hq, hkv, d, "bf16", 25)]
    cos, sin = table(64, 64, "f32", 26)
    pos = torch.arange(n, device=DEV)
    qw, kw = weights(d, "bf16", 27)
    slots = torch.arange(n, device=DEV)
    kp, vp = pools(4, hkv, d, "bf16")

    def step(kp, vp):
        return paged_kv_write_rope(q, k, v, kp, vp, slots, cos, sin, pos, q_weight=qw, k_weight=kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(kp, vp)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(kp, vp)
    for i in range(4):
        q.normal_(generator=torch.Generator(device=DEV).manual_seed(i))
        k.mul_(-1.5)
        pos.add_(7)
        slots.add_(5)
        kr, vr = pools(4, hkv, d, "bf16")
        kp.copy_(kr)
        vp.copy_(vr)
        graph.replay()
        want = step(kr, vr)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(raw(kp), raw(kr)) and torch.equal(raw(vp), raw(vr))
    assert first.shape == out.shape


def test_refusals_on_the_gpu():
    q, k, v = projection(4, 4, 2, 64, "f16", 28)
    cos, sin = table(4, 32, "f32", 29)
    pos = torch.arange(4, device=DEV)
    kp, vp = pools(1, 2, 64, "f16")
    w = torch.ones(64, device=DEV)
    bad = [
        (ValueError, lambda: qk_norm_rope(q, k[:3], cos, sin)),
        (ValueError, lambda: qk_norm_rope(q, k.float(), cos, sin)),
        (ValueError, lambda: qk_norm_rope(q[0], k, cos, sin)),
        (ValueError, lambda: qk_norm_rope(q, k, cos, None)),
        (ValueError, lambda: qk_norm_rope(q, k, cos, sin.half())),
        (ValueError, lambda: qk_norm_rope(q, k, cos[:3], sin[:3])),
        (ValueError, lambda: qk_norm_rope(q, k, None, None, pos)),
        (ValueError, lambda: qk_norm_rope(q, k, cos, sin, pos[:3])),
        (ValueError, lambda: qk_norm_rope(q, k, cos, sin, pos.float())),
        (ValueError, lambda: qk_norm_rope(q, k, torch.cat([cos, cos], 1), torch.cat([sin, sin], 1))),
        (ValueError, lambda: qk_norm_rope(q, k, cos[:0], sin[:0], pos)),
        (ValueError, lambda: qk_norm_rope(q, k, cos, sin, pos, q_weight=w[:32])),
        (ValueError, lambda: qk_norm_rope(q, k, cos, sin, pos, q_weight=w, k_weight=w.half())),
        (ValueError, lambda: qk_norm_rope(q, k, cos, sin, pos, q_weight=w, eps=float("nan"))),
        (NotImplementedError, lambda: qk_norm_rope(q, k, cos[:, :9], sin[:, :9], pos)),
        (NotImplementedError, lambda: qk_norm_rope(q[..., :24], k[..., :24], cos[:, :8], sin[:, :8], pos)),
        (NotImplementedError, lambda: qk_norm_rope(q.double(), k.double(), cos, sin, pos)),
        (RuntimeError, lambda: qk_norm_rope(q, k, cos.cpu(), sin, pos)),
        (RuntimeError, lambda: qk_norm_rope(q.clone().requires_grad_(), k, cos, sin, pos)),
        (RuntimeError, lambda: qk_norm_rope(q, k, cos, sin, pos, q_weight=w.clone().requires_grad_())),
        (ValueError, lambda: paged_kv_write_rope(q, k, v, kp, vp, pos[:3], cos, sin, pos)),
        (ValueError, lambda: paged_kv_write_rope(q, k, v, kp, vp, pos.int(), cos, sin, pos)),
        (ValueError, lambda: paged_kv_write_rope(None, k, v, kp, vp, pos, cos, sin, pos, q_weight=w)),
        (ValueError, lambda: paged_kv_write_rope(q, k, v, kp, vp, pos, cos, sin, pos, k_scale=w[0], v_scale=w[0])),
        (ValueError, lambda: paged_kv_write_rope(q.float(), k, v, kp, vp, pos, cos, sin, pos)),
        (NotImplementedError, lambda: paged_kv_write_rope(q, k, v, kp.float(), vp.float(), pos, cos, sin, pos)),
        (RuntimeError, lambda: paged_kv_write_rope(q, k, v, kp.cpu(), vp.cpu(), pos, cos, sin, pos)),
        (RuntimeError, lambda: paged_kv_write_rope(q, k, v.clone().requires_grad_(), kp, vp, pos, cos, sin, pos)),
    ]
    before = raw(kp).clone()
    for i, (err, call) in enumerate(bad):
        with pytest.raises(err):
            call()
            pytest.fail(f"call {i} was accepted")
    assert torch.equal(raw(kp), before)
    with torch.no_grad():
        qk_norm_rope(q.clone().requires_grad_(), k, cos, sin, pos)
