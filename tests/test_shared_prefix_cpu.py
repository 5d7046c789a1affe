"""Refusals and workspace sizes of the shared-prefix decode's C entry points
(no GPU: arguments are validated before any HIP call)."""
import pytest
import torch

from fasterkernels_amd import native as nat
from fskernels.hip import paged_flash_decode_shared

FAKE = 0x10000  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    return nat.load()


def args(**kw):
    a = dict(q=FAKE, qsb=4096, qsh=128, k=FAKE, kp=16384, kh=2048, kt=128, v=FAKE, vp=16384, vh=2048, vt=128, bt=FAKE,
             bts=64, mb=64, lens=FAKE, shared=512, pages=1000, page=16, sink=None, mode=nat.FSK_SINK_EXP, ks=None,
             vs=None, out=FAKE, osb=4096, osh=128, B=8, hq=32, hkv=8, d=128, qd=nat.FSK_F16, kd=nat.FSK_F16,
             od=nat.FSK_F16, sm=0.1, ws=FAKE, wsb=1 << 40, stream=None)
    assert not set(kw) - set(a), kw
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("override,code", [
    (dict(q=None), "INVALID"), (dict(k=None), "INVALID"), (dict(bt=None), "INVALID"), (dict(lens=None), "INVALID"),
    (dict(out=None), "INVALID"), (dict(shared=-1), "INVALID"), (dict(shared=1025), "INVALID"),
    (dict(shared=1 << 62), "INVALID"), (dict(mb=-1), "UNSUPPORTED"), (dict(bts=63), "INVALID"), (dict(page=24), "UNSUPPORTED"),
    (dict(pages=0), "INVALID"), (dict(hq=33), "INVALID"), (dict(d=96), "UNSUPPORTED"), (dict(B=-1), "INVALID"),
    (dict(B=1 << 20), "UNSUPPORTED"), (dict(kd=nat.FSK_BF16), "UNSUPPORTED"), (dict(kd=nat.FSK_E4M3), "INVALID"),
    (dict(qd=nat.FSK_E4M3, kd=nat.FSK_E4M3, ks=FAKE, vs=FAKE), "UNSUPPORTED"), (dict(od=nat.FSK_E4M3), "UNSUPPORTED"),
    (dict(q=FAKE + 8), "INVALID"), (dict(kt=64), "INVALID"), (dict(sm=float("inf")), "INVALID"), (dict(mode=5), "INVALID"),
    (dict(ws=None), "WORKSPACE"), (dict(ws=FAKE + 16), "WORKSPACE"), (dict(wsb=1000), "WORKSPACE"),
])
def test_refusals(lib, override, code):
    assert lib.fsk_decode_paged_shared(*args(**override)) == getattr(nat, "FSK_ERR_" + code)
    assert lib.fsk_last_error()


def test_workspace(lib):
    f = lib.fsk_shared_workspace_bytes
    need = f(8, 32, 8, 128, 64, 16, 512)
    whole = lib.fsk_workspace_bytes(nat.FSK_LAYOUT_PAGED, 8, 32, 8, 128, 64, 16, 0)
    assert need >= whole  # either way of decoding fits
    # less than a page shared: the paged decode's own workspace
    plain = lib.fsk_workspace_bytes(nat.FSK_LAYOUT_PAGED, 8, 32, 8, 128, 64, 16, 0)
    assert f(8, 32, 8, 128, 64, 16, 15) == plain
    assert f(8, 32, 8, 128, 64, 16, 16) > 0 and f(8, 32, 8, 128, 64, 16, 1024) > 0
    for bad, code in ((dict(shared_len=-1), "INVALID"), (dict(shared_len=1025), "INVALID"),
                      (dict(page_size=24), "UNSUPPORTED"), (dict(head_dim=96), "UNSUPPORTED"),
                      (dict(batch=1 << 20), "UNSUPPORTED"), (dict(num_q_heads=33), "INVALID"),
                      (dict(max_blocks=1 << 40), "UNSUPPORTED")):
        a = dict(batch=8, num_q_heads=32, num_kv_heads=8, head_dim=128, max_blocks=64, page_size=16, shared_len=512)
        a.update(bad)
        assert f(*a.values()) == getattr(nat, "FSK_ERR_" + code), bad
    # the largest batch and table: sizes stay positive
    assert f(16384, 1 << 16, 1, 256, (1 << 17) - 64, 16, 1 << 20) != 0


def test_share_option(lib):
    for bad in (-1, 3):
        assert lib.fsk_set_option(b"share", bad) == nat.FSK_ERR_INVALID
    for ok in (0, 2, 1):
        assert lib.fsk_set_option(b"share", ok) == nat.FSK_OK


def test_empty_batch_needs_no_gpu(lib):
    assert lib.fsk_decode_paged_shared(*args(B=0)) == nat.FSK_OK


def test_host_tensors_are_refused():
    q = torch.zeros(2, 32, 128, dtype=torch.float16)
    pool = torch.zeros(4, 8, 16, 128, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="GPU"):
        paged_flash_decode_shared(q, pool, pool, torch.zeros(2, 2, dtype=torch.int32), torch.tensor([20, 20]), 16, 16)
