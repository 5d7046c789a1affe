"""Refusals of the norm-and-rotation entry points that need no GPU: the C ABI
validates before any HIP call, and the Python entry points reject host tensors."""
import pytest
import torch

from fasterkernels_amd import native as nat
from fskernels.hip import paged_kv_write_rope, qk_norm_rope

FAKE = 0x10000  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    return nat.load()


def rope_args(**kw):
    a = dict(q=FAKE, qst=4096, qsh=128, k=FAKE, kst=1024, ksh=128, n=4, cos=FAKE, cs=64, sin=FAKE, ss=64, rows=100,
             tdt=nat.FSK_F32, rotary=128, inter=0, pos=FAKE, qw=FAKE, kw=FAKE, wdt=nat.FSK_BF16, eps=1e-6, qo=FAKE,
             qost=4096, qosh=128, ko=FAKE, kost=1024, kosh=128, hq=32, hkv=8, d=128, dt=nat.FSK_BF16, stream=None)
    assert not set(kw) - set(a), kw
    a.update(kw)
    return list(a.values())


def write_args(**kw):
    a = dict(q=FAKE, qst=4096, qsh=128, k=FAKE, kst=1024, ksh=128, v=FAKE, vst=1024, vsh=128, slots=FAKE, n=4,
             cos=FAKE, cs=64, sin=FAKE, ss=64, rows=100, tdt=nat.FSK_F32, rotary=128, inter=0, pos=FAKE, qw=FAKE,
             kw=FAKE, wdt=nat.FSK_BF16, eps=1e-6, qo=FAKE, qost=4096, qosh=128, kp=FAKE, kpp=16384, kph=2048, kpt=128,
             vp=FAKE, vpp=16384, vph=2048, vpt=128, pages=10, page=16, hq=32, hkv=8, d=128, dt=nat.FSK_BF16,
             pdt=nat.FSK_BF16, ks=None, vs=None, bt=None, btn=0, upd=None, nupd=0, stream=None)
    assert not set(kw) - set(a), kw
    a.update(kw)
    return list(a.values())


COMMON = [
    (dict(q=None), "INVALID"), (dict(k=None), "INVALID"), (dict(qo=None), "INVALID"), (dict(q=FAKE + 8), "INVALID"),
    (dict(qst=4097), "INVALID"), (dict(ksh=-128), "INVALID"), (dict(kst=1 << 40), "UNSUPPORTED"),
    (dict(n=-1), "INVALID"), (dict(n=1 << 31), "UNSUPPORTED"), (dict(n=(1 << 31) - 1), "UNSUPPORTED"),
    (dict(cos=None), "INVALID"), (dict(sin=None), "INVALID"), (dict(cs=63), "INVALID"), (dict(ss=-64), "INVALID"),
    (dict(rows=0), "INVALID"), (dict(rows=-1), "UNSUPPORTED"), (dict(rows=1 << 31), "UNSUPPORTED"),
    (dict(rows=3, pos=None), "INVALID"), (dict(tdt=nat.FSK_E4M3), "UNSUPPORTED"), (dict(rotary=144), "INVALID"),
    (dict(rotary=-16), "INVALID"), (dict(rotary=24), "UNSUPPORTED"), (dict(wdt=nat.FSK_E4M3), "UNSUPPORTED"),
    (dict(qw=FAKE + 2), "INVALID"), (dict(eps=-1.0), "INVALID"), (dict(eps=float("inf")), "INVALID"),
    (dict(hkv=0), "INVALID"), (dict(hq=-1), "INVALID"), (dict(hq=1 << 20), "UNSUPPORTED"), (dict(d=0), "INVALID"),
    (dict(d=120), "UNSUPPORTED"), (dict(d=512), "UNSUPPORTED"), (dict(dt=nat.FSK_E4M3), "UNSUPPORTED"),
    (dict(dt=17), "UNSUPPORTED"),
]


@pytest.mark.parametrize("override,code", COMMON + [(dict(ko=None), "INVALID"), (dict(kost=1020), "INVALID"),
                                                    (dict(hq=0), "INVALID")])
def test_norm_rope_refuses(lib, override, code):
    assert lib.fsk_qk_norm_rope(*rope_args(**override)) == getattr(nat, "FSK_ERR_" + code)
    assert lib.fsk_last_error()


@pytest.mark.parametrize("override,code", COMMON + [
    (dict(v=None), "INVALID"), (dict(vst=-8), "INVALID"), (dict(slots=None), "INVALID"), (dict(kp=None), "INVALID"),
    (dict(vp=FAKE + 8), "INVALID"), (dict(kpt=64), "INVALID"), (dict(kpt=124), "INVALID"), (dict(pages=0), "INVALID"),
    (dict(page=0), "INVALID"), (dict(pages=1 << 28), "UNSUPPORTED"), (dict(pdt=nat.FSK_F32), "UNSUPPORTED"),
    (dict(ks=FAKE), "INVALID"), (dict(ks=FAKE, vs=FAKE), "INVALID"), (dict(nupd=1), "INVALID"),
    (dict(nupd=-1), "INVALID"), (dict(nupd=1 << 30, bt=FAKE, upd=FAKE, btn=10), "UNSUPPORTED"),
])
def test_write_rope_refuses(lib, override, code):
    assert lib.fsk_paged_write_rope(*write_args(**override)) == getattr(nat, "FSK_ERR_" + code)
    assert lib.fsk_last_error()


def test_nothing_to_do_needs_no_gpu(lib):
    assert lib.fsk_qk_norm_rope(*rope_args(n=0, q=None, k=None, qo=None, ko=None, cos=None, sin=None)) == nat.FSK_OK
    assert lib.fsk_paged_write_rope(*write_args(n=0, q=None, k=None, v=None, slots=None, kp=None, vp=None)) == nat.FSK_OK


def test_host_tensors_are_refused():
    q, k = torch.zeros(2, 4, 64), torch.zeros(2, 2, 64)
    t = torch.zeros(2, 32)
    with pytest.raises(RuntimeError, match="GPU"):
        qk_norm_rope(q, k, t, t)
    pool = torch.zeros(1, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="GPU"):
        paged_kv_write_rope(q, k, k, pool, pool, torch.zeros(2, dtype=torch.long), t, t)
    with pytest.raises(TypeError):
        qk_norm_rope([1], k, t, t)
    with pytest.raises(TypeError):
        paged_kv_write_rope(q, k, k, None, pool, torch.zeros(2, dtype=torch.long), t, t)
