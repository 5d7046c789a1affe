"""GPU parity of the shared-prefix paged decode (paged_flash_decode_shared)
against attention over each sequence's own tokens in float64.

Bar, derived: with p the softmax weights, a value of the output is off by at most
  sum_t p_t |v_t| (e_P + 2 e_s + n 2^-23) + half a step of the output type,
where e_P is P's rounding (f16 2^-11; bf16 hi + lo parts 2^-17), e_s the error of
a score (fp32 sums of D products: (D + 8) 2^-24 times the largest sum |q k| times
the scale, plus the exponential's own 2^-22), and n 2^-23 covers fp32 sums over
the n tokens and f16 weights below the normal range.
"""
import math

import pytest
import torch

from fasterkernels_amd import native as nat
from fskernels.hip import paged_flash_decode, paged_flash_decode_shared
from fskernels.engine import DecodeGraph

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def always_shared():
    """The small batches here on the shared kernels too."""
    nat.set_option("share", 2)
    yield
    nat.set_option("share", 1)


DT = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


class Batch:
    """Sequences of ``lens`` tokens that share their first ``prefix`` (in whole
    pages) on scattered pages of a pool."""

    def __init__(self, lens, prefix, heads, kv, *, page=16, seed=0, sinks=False, extra_blocks=0, q_dtype=None):
        hq, hkv, d = heads
        g = torch.Generator().manual_seed(seed)
        self.lens, self.prefix, self.heads, self.kv, self.page = lens, prefix, heads, kv, page
        B = len(lens)
        common = prefix // page
        need = [max(0, -(-n // page) - common) for n in lens]
        P = common + sum(need) + 3
        perm = torch.randperm(P, generator=g).to(torch.int32)
        table = torch.full((B, common + max(need) + extra_blocks), -1, dtype=torch.int32)
        table[:, :common] = perm[:common]
        off = common
        for b, m in enumerate(need):
            table[b, common:common + m] = perm[off:off + m]
            off += m
        self.table = table.to(DEV)
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        qdt = q_dtype or ("bf16" if kv == "e4m3" else kv)
        self.q = torch.randn(B, hq, d, generator=g).to(DT[qdt]).to(DEV)
        self.k, self.v = (torch.randn(P, hkv, page, d, generator=g).to(DT[kv]).to(DEV) for _ in range(2))
        self.ks = self.vs = None
        if kv == "e4m3":
            self.ks, self.vs = torch.tensor(0.7, device=DEV), torch.tensor(1.3, device=DEV)
        self.sinks = torch.randn(hq, generator=g).to(DEV) if sinks else None

    def rows(self, pool, b, scale):
        n = self.lens[b]
        ids = self.table[b, :-(-n // self.page)].long()
        raw = pool.view(torch.uint8)[ids].view(pool.dtype) if pool.element_size() == 1 else pool[ids]
        x = raw.float().double().transpose(0, 1).reshape(self.heads[1], -1, self.heads[2])[:, :n]
        return x if scale is None else x * scale.double()

    def exact(self, sm=None, mode="exp"):
        """(output, bar's sum p |v| term) in float64."""
        hq, hkv, d = self.heads
        sm = d ** -0.5 if sm is None else sm
        out = torch.zeros(len(self.lens), hq, d, dtype=torch.float64, device=DEV)
        bar = torch.zeros_like(out)
        e_p = 2.0 ** -17 if self.kv == "bf16" else 2.0 ** -11
        for b, n in enumerate(self.lens):
            if n == 0:
                continue
            k, v = self.rows(self.k, b, self.ks), self.rows(self.v, b, self.vs)
            q = self.q[b].double().view(hkv, -1, d)
            x = torch.matmul(q, k.transpose(1, 2).contiguous()) * sm
            top = x.amax(-1, keepdim=True)
            p = torch.exp(x - top)
            den = p.sum(-1, keepdim=True)
            if self.sinks is not None:
                z = self.sinks.double().view(hkv, -1, 1)
                den = den + (torch.exp(z - top) if mode == "exp" else z)
            p = p / den
            out[b] = torch.matmul(p, v).view(hq, d)
            mag = torch.matmul(q.abs(), k.abs().transpose(1, 2).contiguous()).amax() * abs(sm)
            e_s = (d + 8) * 2.0 ** -24 * mag.item() + 2.0 ** -22
            bar[b] = torch.matmul(p.abs(), v.abs()).view(hq, d) * (e_p + 2 * e_s + n * 2.0 ** -23)
        return out, bar

    def run(self, **kw):
        kw.setdefault("sink_mode", "exp")
        return paged_flash_decode_shared(self.q, self.k, self.v, self.table, self.seq_lens, self.page, self.prefix,
                                         s_aux=self.sinks, k_scale=self.ks, v_scale=self.vs, **kw)

    def plain(self, **kw):
        kw.setdefault("sink_mode", "exp")
        return paged_flash_decode(self.q, self.k, self.v, self.table, self.seq_lens, self.page, s_aux=self.sinks,
                                  k_scale=self.ks, v_scale=self.vs, **kw)


def check(batch, out, what, sm=None, mode="exp"):
    want, bar = batch.exact(sm, mode)
    tol = bar * (1 + 2.0 ** -6) + want.abs() * torch.finfo(out.dtype).eps / 2 + 1e-7
    err = (out.double() - want).abs()
    assert (err <= tol).all(), f"{what}: worst {(err / tol).max().item():.3f} of the bar"


CASES = [
    # lens (after the prefix; None: a spread), batch, prefix, heads, kv, page, sinks
    (1, 16, (8, 8, 128), "f16", 16, False),
    (1, 640, (32, 8, 128), "f16", 16, True),
    (3, 64, (32, 8, 128), "bf16", 16, False),
    (4, 1024, (32, 8, 128), "f16", 16, False),
    (8, 2100, (32, 8, 128), "bf16", 16, True),      # 32 rows a head; a prompt that ends inside a page
    (9, 530, (32, 8, 128), "e4m3", 16, True),       # 36: two waves
    (17, 333, (32, 8, 128), "f16", 32, False),      # 68: four waves, pages of 32
    (70, 700, (16, 8, 128), "e4m3", 16, False),
    (33, 1500, (32, 4, 128), "bf16", 48, True),     # 264 rows, odd pages
    (5, 900, (64, 8, 64), "f16", 16, True),
    (21, 900, (64, 8, 64), "bf16", 16, False),
    (13, 777, (32, 8, 64), "e4m3", 64, True),
    (2, 500, (32, 8, 256), "bf16", 16, False),
    (11, 1200, (32, 8, 256), "f16", 16, True),
    (20, 600, (16, 8, 256), "e4m3", 16, True),
    (6, 800, (32, 1, 128), "f16", 16, False),       # one KV head, 32 query heads each
    (7, 800, (40, 8, 128), "bf16", 16, True),       # five query heads a KV head
]


@pytest.mark.parametrize("B,prefix,heads,kv,page,sinks", CASES)
def test_against_float64(B, prefix, heads, kv, page, sinks):
    g = torch.Generator().manual_seed(B + prefix)
    lens = [prefix + int(n) for n in torch.randint(0, 150, (B,), generator=g)]
    batch = Batch(lens, prefix, heads, kv, page=page, seed=B, sinks=sinks)
    check(batch, batch.run(), "shared")
    check(batch, batch.run(out_dtype=torch.float32), "f32 output")


@pytest.mark.parametrize("heads,kv", [((32, 8, 128), "f16"), ((32, 8, 128), "bf16"), ((64, 8, 64), "e4m3"),
                                      ((32, 8, 256), "bf16")])
def test_short_and_empty_rows(heads, kv):
    """Rows that end inside the prefix, at its ends, or are empty; what lies past
    a row's end (infinities and NaN among it) does not reach it."""
    prefix = 320
    lens = [prefix + 40, 1, 15, 16, 17, 63, 64, 65, 100, 129, 250, 319, 320, 321, 0, prefix + 7, 64, 100]
    batch = Batch(lens, prefix, heads, kv, seed=5, sinks=True)
    check(batch, batch.run(), "short rows")
    # no token of the rows that end before 200 holds these
    page = batch.table[0, 13].item()
    bad = batch.v if kv != "e4m3" else batch.v.view(torch.uint8)
    bad[page, :, 3:5, 1:9] = float("inf") if kv != "e4m3" else 0x7F
    bad[page, 0, 7, 2] = float("nan") if kv != "e4m3" else 0x7F
    kbad = batch.k if kv != "e4m3" else batch.k.view(torch.uint8)
    kbad[page, 0, 9, 2] = float("nan") if kv != "e4m3" else 0x7F
    out = batch.run()
    keep = [b for b, n in enumerate(lens) if n < 200]
    clean = Batch(lens, prefix, heads, kv, seed=5, sinks=True).run()
    assert torch.equal(out[keep], clean[keep])
    assert out[[b for b, n in enumerate(lens) if n > 220]].isnan().any()


def test_empty_rows_follow_the_paged_decode():
    batch = Batch([0, 400, 0, 20], 320, (32, 8, 128), "f16", seed=6)
    a, b = batch.run(), batch.plain()
    assert torch.equal(a.isnan(), b.isnan())
    batch.seq_lens[1:] = torch.tensor([-5, 0, 0])  # a batch without any token
    assert torch.equal(batch.run().isnan(), batch.plain().isnan())


@pytest.mark.parametrize("mode", ["linear", "exp"])
def test_sink_modes_and_scales(mode):
    batch = Batch([300, 290, 256, 411], 256, (32, 8, 128), "f16", seed=7, sinks=True)
    batch.sinks *= 0.1
    for sm in (None, 0.02, -0.05, 0.0):
        check(batch, batch.run(sink_mode=mode, sm_scale=sm), f"{mode} {sm}", sm, mode)


def test_large_scores_and_late_maxima():
    """Scores that grow along the prefix by far more than the lazy maximum's 2^8,
    and weights that all but vanish."""
    batch = Batch([1100] * 6, 1024, (32, 8, 128), "f16", seed=8)
    order = batch.table[0, :64].long()
    for i in range(0, 64, 4):
        batch.k[order[i:i + 4]] *= 0.25 + 0.1 * i
    batch.q *= 3
    check(batch, batch.run(), "growing scores")


def test_linear_sink_counts_against_the_true_maximum():
    """Maxima that grow within the lazy maximum's 2^8, and sinks that show it."""
    batch = Batch([1030] * 5, 1024, (32, 8, 128), "f16", seed=20, sinks=True)
    order = batch.table[0, :64].long()
    for i in range(64):
        batch.k[order[i]] *= 0.2 + 0.01 * i
    batch.sinks.uniform_(20, 60)
    check(batch, batch.run(sink_mode="linear"), "linear sinks", None, "linear")


def test_prefix_of_nothing_and_of_everything():
    batch = Batch([33, 20, 7], 0, (32, 8, 128), "f16", seed=9)
    for shared in (0, 15):  # less than a page: the paged decode itself
        batch.prefix = shared
        assert torch.equal(batch.run(), batch.plain())
    batch = Batch([64, 64, 64], 64, (32, 8, 128), "bf16", seed=10)  # nothing of their own
    check(batch, batch.run(), "prefix only")
    batch = Batch([64, 50, 64], 64, (32, 8, 128), "bf16", seed=10, extra_blocks=40)
    check(batch, batch.run(), "a wide table")


def test_long_own_parts_and_many_rows():
    """Own parts that the split kernel cuts into many partials, and a batch large
    enough for the many-row reduce."""
    batch = Batch([96 + n for n in (4000, 1, 2500, 0)], 96, (32, 8, 128), "f16", seed=11)
    check(batch, batch.run(), "long own parts")
    batch = Batch([160 + n % 50 for n in range(150)], 160, (32, 8, 128), "bf16", seed=12)
    check(batch, batch.run(), "many rows")


def test_long_prefix_and_page_windows():
    """A prefix of many tiles per item (page ids are read 64 at a time)."""
    batch = Batch([20000 + i for i in range(2)], 20000, (8, 8, 128), "bf16", seed=13)
    check(batch, batch.run(), "20000 tokens")
    batch = Batch([9000 + i for i in range(40)], 9000, (16, 1, 64), "f16", seed=14)
    check(batch, batch.run(), "9000 tokens, one KV head")


def test_pool_order_strides_and_bad_pages():
    """Pools with the page dimension inside (a layer's view of a joint tensor), a
    wider query, and table entries outside the pool past the sequences' ends."""
    batch = Batch([300, 280, 310], 256, (32, 8, 128), "f16", seed=15, extra_blocks=3)
    want = batch.run()
    both = torch.stack([batch.k, batch.v], dim=2)  # [P, Hkv, 2, page, D]
    batch.k, batch.v = both[:, :, 0], both[:, :, 1]
    wide = torch.zeros(3, 32, 256, dtype=torch.float16, device=DEV)
    wide[..., :128] = batch.q
    batch.q = wide[..., :128]
    batch.table[:, -2:] = 1 << 30
    assert torch.equal(batch.run(), want)
    batch.seq_lens = batch.seq_lens.cpu()  # host lengths
    assert torch.equal(batch.run(), want)
    batch.seq_lens = batch.seq_lens.long().to(DEV)
    assert torch.equal(batch.run(), want)


def test_repeats_are_bit_identical_and_graphs_follow_their_inputs():
    batch = Batch([700 + 3 * i for i in range(12)], 640, (32, 8, 128), "bf16", seed=16, extra_blocks=4)
    first = batch.run()
    assert torch.equal(first, batch.run())
    graph = DecodeGraph(batch.run)
    for i in range(4):
        batch.q.normal_(generator=torch.Generator(device=DEV).manual_seed(i))
        batch.seq_lens.add_(2)
        got = graph.replay().clone()
        want = batch.run()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = batch.run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, batch.run())


def test_two_calls_at_once():
    a = Batch([700 + i for i in range(16)], 640, (32, 8, 128), "f16", seed=17)
    b = Batch([900 + i for i in range(9)], 512, (64, 8, 64), "bf16", seed=18)
    wa, wb = a.run(), b.run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, x in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(x.run())
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert torch.equal(out, (wa, wb)[i % 2])


def test_which_calls_share():
    """By the rule a small call is the paged decode's own, bit for bit, and a large one
    is not; more sequences than the kernel takes are always the paged decode's."""
    small = Batch([300 + i for i in range(4)], 256, (32, 8, 128), "f16", seed=21)
    large = Batch([2100 + i for i in range(12)], 2048, (32, 8, 128), "f16", seed=22)
    many = Batch([40 + i % 9 for i in range(501)], 32, (8, 1, 64), "f16", seed=23)
    forced = small.run(), large.run()
    assert torch.equal(many.run(), many.plain())
    nat.set_option("share", 1)
    assert torch.equal(small.run(), small.plain()) and not torch.equal(small.run(), forced[0])
    assert torch.equal(large.run(), forced[1]) and not torch.equal(large.run(), large.plain())
    check(large, large.run(), "large")
    nat.set_option("share", 0)
    assert torch.equal(large.run(), large.plain())


def test_refusals():
    batch = Batch([70, 80], 64, (32, 8, 128), "f16", seed=19)

    def call(**kw):
        a = dict(q=batch.q, k=batch.k, v=batch.v, table=batch.table, lens=batch.seq_lens, page=16, shared=64)
        extra = {k: kw.pop(k) for k in list(kw) if k not in a}
        a.update(kw)
        return paged_flash_decode_shared(a["q"], a["k"], a["v"], a["table"], a["lens"], a["page"], a["shared"], **extra)

    for err, kw in [(ValueError, dict(shared=-1)), (ValueError, dict(shared=16 * batch.table.shape[1] + 1)),
                    (ValueError, dict(page=32)), (ValueError, dict(table=batch.table[:1])),
                    (ValueError, dict(lens=batch.seq_lens[:1])), (ValueError, dict(v=batch.v[:, :4])),
                    (ValueError, dict(v=batch.v.bfloat16())), (ValueError, dict(sink_mode="soft")),
                    (ValueError, dict(sm_scale=float("nan"))), (ValueError, dict(s_aux=torch.zeros(3, device=DEV))),
                    (NotImplementedError, dict(q=batch.q.bfloat16())), (NotImplementedError, dict(q=batch.q.float())),
                    (ValueError, dict(k=batch.k.to(torch.float8_e4m3fn), v=batch.v.to(torch.float8_e4m3fn))),
                    (RuntimeError, dict(table=batch.table.cpu())), (RuntimeError, dict(k=batch.k.cpu())),
                    (RuntimeError, dict(q=batch.q.clone().requires_grad_()))]:
        with pytest.raises(err):
            call(**kw)
            pytest.fail(f"{kw} was accepted")
    assert call(q=batch.q[:0]).shape == (0, 32, 128)
