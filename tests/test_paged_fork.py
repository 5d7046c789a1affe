"""Forked sequences of PagedKVCache (host bookkeeping, on host pools): shared pages,
copies of begun pages, holders, and what a batch has in common."""
import random

import pytest
import torch

from fskernels.paged_attn import PAGE_SIZE, PagedKVCache


def cache(num_pages=40, max_seqs=6, dtype=torch.float16, **kw):
    return PagedKVCache(2, num_pages, max_seqs, 12, 2, 8, dtype, "cpu", **kw)


def fill(c, sid, n, value):
    for layer_rows in range(n):
        slots = c.reserve_slots([sid], 1)
        for layer in range(c.num_layers):
            x = torch.full((1, 2, 8), float(value + layer_rows))
            c.write_kv(layer, x, -x, slots)


def tokens(c, sid, layer=0):
    """The values that a sequence's rows hold, in order."""
    n = c._seq_lens[sid]
    table = c.block_table[sid]
    return [c.k_pool[layer, table[t // PAGE_SIZE], 0, t % PAGE_SIZE, 0].float().item() for t in range(n)]


@pytest.mark.parametrize("length", [0, 5, 16, 37, 48])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float8_e4m3fn])
def test_fork_shares_full_pages_and_copies_the_begun_one(length, dtype):
    c = cache(dtype=dtype)
    a = c.allocate_sequence()
    fill(c, a, length, 1)
    before = c.pages_used
    ids = c.fork_sequence(a, 3)
    assert len(set(ids + [a])) == 4
    full, rest = divmod(length, PAGE_SIZE)
    assert c.pages_used == before + (3 if rest else 0)
    assert c.shared_prefix_len([a] + ids) == full * PAGE_SIZE
    want = tokens(c, a)
    for sid in ids:
        assert tokens(c, sid) == want and tokens(c, sid, 1) == want
    # each grows by itself
    for i, sid in enumerate([a] + ids):
        fill(c, sid, 20, 8 * (i + 1))
    got = [tokens(c, sid) for sid in [a] + ids]
    assert all(g[:length] == want for g in got) and len({tuple(g) for g in got}) == 4
    assert c.shared_prefix_len([a] + ids) == full * PAGE_SIZE
    for sid in [ids[1], a, ids[0], ids[2]]:
        assert tokens(c, sid) == got[([a] + ids).index(sid)]
        c.free_sequence(sid)
    assert c.pages_used == 0 and sorted(c._free_pages) == list(range(40)) and not any(c._holders)


def test_shared_prefix_len_of_unlike_sequences():
    c = cache()
    a = c.allocate_sequence()
    fill(c, a, 40, 1)
    b, d = c.fork_sequence(a, 2)
    other = c.allocate_sequence()
    fill(c, other, 40, 1)
    assert c.shared_prefix_len([]) == 0
    assert c.shared_prefix_len([a]) == 32
    assert c.shared_prefix_len([a, b, d]) == c.shared_prefix_len([d, a]) == 32
    assert c.shared_prefix_len([a, other]) == 0
    fill(c, b, 30, 2)
    e, = c.fork_sequence(b)
    assert c.shared_prefix_len([b, e]) == 64 and c.shared_prefix_len([a, e]) == 32


def test_refused_forks_change_nothing():
    c = cache(num_pages=4, max_seqs=4)
    a = c.allocate_sequence()
    fill(c, a, 40, 1)

    def state():
        return (list(c._free_pages), list(c._seq_lens), list(c._active), [list(p) for p in c._pages], list(c._holders),
                c.block_table.tolist())

    before = state()
    with pytest.raises(RuntimeError, match="pages"):
        c.fork_sequence(a, 2)   # one free page, two begun pages wanted
    with pytest.raises(RuntimeError, match="slots"):
        c.fork_sequence(a, 4)
    with pytest.raises(ValueError):
        c.fork_sequence(3)
    with pytest.raises(ValueError):
        c.fork_sequence(-1)
    with pytest.raises(ValueError):
        c.fork_sequence(a, -1)
    assert c.fork_sequence(a, 0) == [] and state() == before
    b, = c.fork_sequence(a)
    with pytest.raises(RuntimeError):  # no page left for an append past the shared ones
        for _ in range(20):
            c.append_kv(a, 0, torch.zeros(1, 2, 1, 8), torch.zeros(1, 2, 1, 8))
    c.free_sequence(a)
    assert tokens(c, b)[:40] == [float(i + 1) for i in range(40)]


def test_random_scripts_keep_the_books():
    rnd = random.Random(5)
    c = cache(num_pages=60, max_seqs=8)
    content = {}
    for step in range(400):
        live = list(content)
        op = rnd.random()
        try:
            if op < 0.15 or not live:
                content[c.allocate_sequence()] = []
            elif op < 0.3:
                s = rnd.choice(live)
                for sid in c.fork_sequence(s, rnd.randint(1, 2)):
                    content[sid] = list(content[s])
            elif op < 0.45:
                s = rnd.choice(live)
                c.free_sequence(s)
                del content[s]
            else:
                s, n = rnd.choice(live), rnd.randint(1, 20)
                fill(c, s, n, step)
                content[s] += [float(step + i) for i in range(n)]
        except (RuntimeError, IndexError):
            for s in live:  # a fill that stopped half way
                content[s] = tokens(c, s)
        held = [0] * 60
        for s in content:
            assert tokens(c, s) == [torch.tensor(v).half().item() for v in content[s]]
            for pp in c._pages[s]:
                held[pp] += 1
        assert held == c._holders
        assert sorted(c._free_pages) == [pp for pp in range(60) if held[pp] == 0]


def test_positions_of_reserved_slots():
    c = cache()
    a, b = c.allocate_sequence(), c.allocate_sequence()
    fill(c, a, 3, 1)
    slots, pos = c.reserve_slots([a, b, a], 2, return_positions=True)
    assert pos.tolist() == [3, 4, 0, 1, 5, 6] and slots.numel() == 6
    assert c.reserve_slots([b], 1).tolist() == [c._pages[b][0] * PAGE_SIZE + 2]
    with pytest.raises(RuntimeError, match="GPU"):
        c.write_qkv_rope(0, None, torch.zeros(1, 2, 8), torch.zeros(1, 2, 8), slots[:1], pos[:1], None, None)
