"""The rotation, the cache write and the shared-prefix decode together, as a
serving loop uses them (PagedKVCache, PagedDecodeStep, the rotary patch).

Bars: stored and returned rows against the rotation's formula in float64, and the
attention against float64 over those rows (each operator's own bars, in
test_gpu_rope and test_gpu_shared_prefix); captured steps against the eager calls
bit for bit.
"""
import pytest
import torch

from fasterkernels_amd import native as nat
from fskernels.engine import PagedDecodeStep
from fskernels.hip import hf as H
from fskernels.hip import paged_flash_decode_shared, paged_kv_write_rope, qk_norm_rope
from fskernels.paged_attn import PAGE_SIZE, PagedKVCache

from .test_gpu_rope import DT, close, oracle, projection, table, weights
from .test_gpu_shared_prefix import Batch, check

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(params=[1, 2], ids=["rule", "always"])
def share(request):
    nat.set_option("share", request.param)
    yield
    nat.set_option("share", 1)


def new_cache(kv, hkv, d, **kw):
    scales = dict(k_scale=0.05, v_scale=0.05) if kv == "e4m3" else {}
    return PagedKVCache(2, 400, 40, 64, hkv, d, DT[kv], DEV, **scales, **kw)


def as_batch(cache, layer, ids, q, kv, sinks):
    b = Batch.__new__(Batch)
    b.lens, b.heads, b.kv, b.page = [cache._seq_lens[s] for s in ids], (q.shape[1], *cache.k_pool.shape[2::2]), kv, 16
    b.table, b.q, b.k, b.v = cache.get_block_table_tensor(ids), q, cache.k_pool[layer], cache.v_pool[layer]
    b.ks, b.vs, b.sinks = cache.k_scale, cache.v_scale, sinks
    return b


@pytest.mark.parametrize("kv,heads,prompt,n", [("f16", (32, 8, 128), 301, 9), ("bf16", (16, 4, 64), 64, 20),
                                               ("e4m3", (32, 8, 128), 530, 5), ("bf16", (8, 2, 256), 95, 3)])
def test_prompt_fork_and_steps(kv, heads, prompt, n, share):
    """A prompt stored, n samples forked from it, six steps of each."""
    hq, hkv, d = heads
    src = "bf16" if kv == "e4m3" else kv
    cache = new_cache(kv, hkv, d)
    cos, sin = table(1024, d // 2, "f32", 1)
    qw, kw = weights(d, src, 2)
    sinks = torch.randn(hq, generator=torch.Generator().manual_seed(3)).to(DEV)
    opts = dict(q_weight=qw, k_weight=kw, eps=1e-6)

    def store(ids, tokens, seed):
        q, k, v = projection(len(ids) * tokens, hq, hkv, d, src, seed)
        slots, pos = cache.reserve_slots(ids, tokens, return_positions=True)
        for layer in range(2):
            out = cache.write_qkv_rope(layer, q, k, v, slots, pos, cos, sin, **opts)
            close(out, *oracle(q, qw, cos, sin, pos, 1e-6, False), src, "queries")
            want, mag = oracle(k, kw, cos, sin, pos, 1e-6, False)
            rows = cache.k_pool[layer].float()[slots // 16, :, slots % 16]
            s = float(cache.k_scale) if kv == "e4m3" else 1.0
            if kv == "e4m3":  # codes of x / scale, clamped; 2 more fp32 roundings in the quotient
                want, mag = (want / s).clamp(-448, 448), mag / s
                mag = mag * (20 / 18)
            close(rows, want, mag, kv, "keys")
        return out

    first = cache.allocate_sequence()
    store([first], prompt, 10)
    ids = [first] + cache.fork_sequence(first, n - 1)
    prefix = cache.shared_prefix_len(ids)
    assert prefix == (prompt // PAGE_SIZE * PAGE_SIZE if n > 1 else cache._seq_lens[first] // 16 * 16)
    for t in range(6):
        q = store(ids, 1, 20 + t)
        batch = as_batch(cache, 1, ids, q, kv, sinks)
        out = paged_flash_decode_shared(q, batch.k, batch.v, batch.table, cache.get_seq_lens_tensor(ids), 16, prefix,
                                        s_aux=sinks, k_scale=batch.ks, v_scale=batch.vs, sink_mode="exp")
        check(batch, out, f"step {t}")
    for sid in ids:
        cache.free_sequence(sid)
    assert cache.pages_used == 0


@pytest.mark.parametrize("kv,inter", [("f16", False), ("e4m3", True)])
def test_captured_step_with_rotation_and_shared_prefix(kv, inter, share):
    hq, hkv, d, n = 32, 8, 128, 8
    src = torch.bfloat16 if kv == "e4m3" else DT[kv]
    cos, sin = table(200, d // 2, "f32", 4)
    qw, kw = weights(d, "f32", 5)
    sinks = torch.randn(hq, generator=torch.Generator().manual_seed(6)).to(DEV)
    rope = dict(q_weight=qw, k_weight=kw, eps=1e-5, interleaved=inter)
    g = torch.Generator().manual_seed(7)

    def rows(tokens, heads):
        return torch.randn(tokens, heads, d, generator=g).to(src).to(DEV)

    caches = [new_cache(kv, hkv, d) for _ in range(2)]
    prompt = rows(150, hkv), rows(150, hkv)
    for c in caches:
        a = c.allocate_sequence()
        slots, pos = c.reserve_slots([a], 150, return_positions=True)
        c.write_qkv_rope(1, None, *prompt, slots, pos, cos, sin, k_weight=kw, eps=1e-5, interleaved=inter)
        ids = [a] + c.fork_sequence(a, n - 1)
    cache, twin = caches
    step = PagedDecodeStep(cache, 1, ids, hq, s_aux=sinks, sink_mode="exp", rope=(cos, sin), share_prefix=True, **rope)
    assert step.shared_len == 144
    for t in range(50):
        q, k, v = rows(n, hq), rows(n, hkv), rows(n, hkv)
        out = step.step(q, k, v)
        torch.cuda.synchronize()
        slots, pos = twin.reserve_slots(ids, 1, return_positions=True)
        qr = twin.write_qkv_rope(1, q, k, v, slots, pos, cos, sin, **rope)
        want = paged_flash_decode_shared(qr, twin.k_pool[1], twin.v_pool[1], twin.get_block_table_tensor(ids),
                                         twin.get_seq_lens_tensor(ids), 16, 144, s_aux=sinks, k_scale=twin.k_scale,
                                         v_scale=twin.v_scale, sink_mode="exp")
        torch.cuda.synchronize()
        assert torch.equal(out, want), t
        assert torch.equal(cache.block_table, twin.block_table), t
    assert torch.equal(cache.k_pool.view(torch.uint8), twin.k_pool.view(torch.uint8))
    check(as_batch(twin, 1, ids, qr, kv, sinks), out, "last step")
    # all 200 rows of the tables are used up: refused before anything changes
    lens = list(cache._seq_lens)
    with pytest.raises(IndexError, match="200"):
        step.step(q, k, v)
    assert cache._seq_lens == lens


def test_captured_step_refuses_a_prefix_that_is_gone():
    cache = new_cache("f16", 8, 128)
    a = cache.allocate_sequence()
    cache.reserve_slots([a], 64)
    ids = [a] + cache.fork_sequence(a, 2)
    step = PagedDecodeStep(cache, 0, ids, 32, share_prefix=True)
    other = cache.allocate_sequence()
    cache.free_sequence(other)
    step.step()                      # freeing another sequence is no matter
    cache.free_sequence(ids[1])
    assert cache.allocate_sequence() == ids[1]
    cache.reserve_slots([ids[1]], 64)
    lens = list(cache._seq_lens)
    with pytest.raises(RuntimeError, match="share"):
        step.step()
    assert cache._seq_lens == lens
    normed = PagedDecodeStep(cache, 0, ids, 32, rope=(None, None), k_weight=torch.ones(128, device=DEV).half())
    normed.step(k_new=torch.full((3, 8, 128), 2.0, device=DEV).half())
    torch.cuda.synchronize()
    page = cache._pages[ids[0]][(cache._seq_lens[ids[0]] - 1) // 16]
    assert (cache.k_pool[0, page, :, (cache._seq_lens[ids[0]] - 1) % 16] == 1).all()  # 2 / sqrt(4 + 1e-6), rounded
    with pytest.raises(ValueError, match="rope"):
        PagedDecodeStep(cache, 0, ids, 32, q_weight=torch.ones(128, device=DEV))


@pytest.mark.parametrize("kv", ["f16", "e4m3"])
def test_forked_begun_page_is_a_copy_on_the_device(kv):
    cache = new_cache(kv, 2, 64)
    a = cache.allocate_sequence()
    k = torch.randn(21, 2, 64, generator=torch.Generator().manual_seed(8)).to(DEV)
    slots = cache.reserve_slots([a], 21)
    cache.write_kv(1, k, -k, slots)
    b, c = cache.fork_sequence(a, 2)
    rows = cache.get_block_table_tensor([a, b, c]).long().cpu()
    assert (rows[:, 0] == rows[0, 0]).all() and len(set(rows[:, 1].tolist())) == 3
    for pool in (cache.k_pool, cache.v_pool):
        raw = pool.view(torch.uint8).cpu()
        for other in rows[1:, 1]:
            assert torch.equal(raw[:, other, :, :5], raw[:, rows[0, 1], :, :5])


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("batch,tables,seq", [(1, 1, 1), (3, 3, 1), (3, 1, 17), (2, 2, 33)])
def test_rotary_patch(dt, batch, tables, seq):
    g = torch.Generator().manual_seed(seq)
    cos, sin = table(tables * seq, 32, dt, 9)
    wide = [torch.cat([t, t], 1).view(tables, seq, 64) for t in (cos, sin)]
    # (as a model holds them: the heads of a projection, seen as [B, H, S, D])
    q, k = (torch.randn(batch, seq, h, 64, generator=g).to(DT[dt]).to(DEV).transpose(1, 2) for h in (6, 2))
    called = []
    fn = H.hf_rotary(lambda *a, **kw: called.append(1))
    qo, ko = fn(q, k, *wide)
    row = torch.arange(batch * seq) % (tables * seq)
    assert not called
    for got, x in ((qo, q), (ko, k)):
        assert got.shape == x.shape and got.dtype is x.dtype
        flat = x.transpose(1, 2).reshape(batch * seq, -1, 64)
        close(got.transpose(1, 2).reshape(flat.shape), *oracle(flat, None, cos, sin, row, 0, False), dt, "patch")
    # calls that the kernel does not take
    fn(q, k, *wide, unsqueeze_dim=2)
    fn(q, k, wide[0][..., :32], wide[1][..., :32])
    fn(q.clone().requires_grad_(), k, *wide)
    fn(q.transpose(1, 2), k.transpose(1, 2), *wide, 2)
    assert len(called) == 4
    with torch.no_grad():
        fn(q.clone().requires_grad_(), k, *wide)
    assert len(called) == 4


def test_model_runs_through_the_rotary_patch():
    """Prompt and steps of a float32 model with and without the patch."""
    transformers = pytest.importorskip("transformers")
    import transformers.models.qwen3.modeling_qwen3 as qm
    cfg = transformers.Qwen3Config(vocab_size=256, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                                   num_attention_heads=8, num_key_value_heads=2, head_dim=128,
                                   max_position_embeddings=512, attn_implementation="eager")
    torch.manual_seed(0)
    model = transformers.Qwen3ForCausalLM(cfg).to(DEV, torch.float32).eval()
    ids = torch.randint(0, 256, (2, 24), generator=torch.Generator().manual_seed(1)).to(DEV)
    calls = []

    def logits():
        with torch.no_grad():
            out = model(ids[:, :20], use_cache=True)
            got = [out.logits]
            for t in range(20, 24):
                out = model(ids[:, t:t + 1], past_key_values=out.past_key_values, use_cache=True)
                got.append(out.logits)
        return torch.cat(got, 1)

    before = qm.apply_rotary_pos_emb
    want = logits()
    with H.patched_hf_rotary():
        inner = qm.apply_rotary_pos_emb

        def spy(*a, **kw):
            calls.append(H._kernel_rotates(*a[:4]))
            return inner(*a, **kw)

        qm.apply_rotary_pos_emb = spy
        got = logits()
    assert qm.apply_rotary_pos_emb is before
    assert calls == [True] * (2 * 5)
    # fp32 throughout: the two differ by roundings of 2^-24 relative in the rotated rows,
    # which two layers of this width carry on (sums of at most 1024 products each)
    assert (got - want).abs().max() <= 1024 * 2.0 ** -24 * 16 * want.abs().max()


# ---------------------------------------------------------------------------
def table_of(rows, d):
    return table(rows, d // 2, "f32", 13)


def test_pools_past_four_gigabytes(share):
    """Pages behind 2^32 bytes of a layer's pool, shared and own, written and read."""
    P, hq, hkv, d, n = 140000, 32, 8, 128, 6
    k_pool, v_pool = (torch.empty(P, hkv, 16, d, dtype=torch.float16, device=DEV) for _ in range(2))
    assert k_pool.numel() * 2 > 1 << 32
    g = torch.Generator().manual_seed(11)
    prefix, lens = 256, [300 + 7 * i for i in range(n)]
    shared = torch.cat([torch.arange(8), torch.arange(P - 8, P)])
    own = torch.cat([torch.arange(8, 8 + 5 * n), torch.arange(P - 8 - 5 * n, P - 8)]).view(2, n, 5)
    table = torch.cat([shared.expand(n, 16), own[1], own[0]], 1).int().to(DEV)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=DEV)
    used = table.long().unique()
    k_pool[used] = torch.randn(len(used), hkv, 16, d, generator=g).half().to(DEV)
    v_pool[used] = torch.randn(len(used), hkv, 16, d, generator=g).half().to(DEV)
    # the last token of every sequence through the writing rotation
    q, k, v = projection(n, hq, hkv, d, "f16", 12)
    cos, sin = table_of(400, d)
    at = lens_t.long() - 1
    slots = table.gather(1, (at // 16)[:, None]).long()[:, 0] * 16 + at % 16
    assert (slots * hkv * d * 2 > 1 << 32).all()
    qr = paged_kv_write_rope(q, k, v, k_pool, v_pool, slots, cos, sin, at)
    close(k_pool[slots // 16, :, slots % 16], *oracle(k, None, cos, sin, at, 0, False), "f16", "keys")
    assert torch.equal(v_pool[slots // 16, :, slots % 16], v)
    out = paged_flash_decode_shared(qr, k_pool, v_pool, table, lens_t, 16, prefix)
    b = Batch.__new__(Batch)
    b.lens, b.heads, b.kv, b.page, b.table, b.q, b.k, b.v = lens, (hq, hkv, d), "f16", 16, table, qr, k_pool, v_pool
    b.ks = b.vs = b.sinks = None
    check(b, out, "far pages")


def test_rows_past_four_gigabytes():
    step = 1_200_000_000
    base = torch.empty(2 * step + 8192, dtype=torch.bfloat16, device=DEV)
    q = base.as_strided((3, 32, 128), (step, 128, 1))
    k = base[4096:].as_strided((3, 8, 128), (step, 128, 1))
    q.copy_(torch.randn(3, 32, 128, generator=torch.Generator().manual_seed(14)))
    k.copy_(torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(15)))
    cos, sin = table_of(3, 128)
    qo, ko = qk_norm_rope(q, k, cos, sin)
    row = torch.arange(3)
    close(qo, *oracle(q, None, cos, sin, row, 0, False), "bf16", "queries")
    close(ko, *oracle(k, None, cos, sin, row, 0, False), "bf16", "keys")


@pytest.mark.parametrize("kv", ["f16", "e4m3"])
def test_fork_in_a_cache_past_four_gigabytes(kv):
    P = 140000 if kv == "f16" else 280000
    cache = PagedKVCache(2, P, 8, 8, 8, 128, DT[kv], DEV)
    assert cache.k_pool[0].numel() * cache.k_pool.element_size() > 1 << 32
    a = cache.allocate_sequence()
    g = torch.Generator().manual_seed(16)
    slots = cache.reserve_slots([a], 21)
    for layer in range(2):
        cache.write_kv(layer, *(torch.randn(21, 8, 128, generator=g).to(DEV) for _ in range(2)), slots)
    b, c = cache.fork_sequence(a, 2)
    old, *new = [cache._pages[s][1] for s in (a, b, c)]
    for pool in (cache.k_pool, cache.v_pool):
        for layer in range(2):
            want = pool[layer, old].float()
            assert want[:, :5].any()
            for page in new:
                assert torch.equal(pool[layer, page].float(), want)
        assert not pool[0, min(new) - 1].float().any()  # its neighbour is as it was
