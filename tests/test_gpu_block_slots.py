"""Block tables and slot maps built on the GPU, against the same pool kept on the host."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from oracle import fp8_cache as of
from qwenquest_amd.paged import BlockReqToTokenPool

pytestmark = pytest.mark.gpu


def i64(x, dev):
    return torch.tensor(x, dtype=torch.int64, device=dev)


def check(pool, want, loc=None, pos=None, got=None):
    if got is not None:
        assert np.array_equal(got[0].cpu().numpy(), loc)
        assert np.array_equal(got[1].cpu().numpy(), pos)
    assert pool.held.tolist() == [len(t) for t in want.table]
    table = pool.block_table.cpu().numpy()
    for r, t in enumerate(want.table):
        assert table[r, : len(t)].tolist() == t and not table[r, len(t) :].any()
    assert np.array_equal(pool.req_to_token.cpu().numpy(), want.r2t)
    n = int(pool.free_count)
    assert pool.free_blocks[:n].tolist() == want.stack


@pytest.mark.parametrize("seed", range(6))
def test_a_server_s_life(cuda, seed):
    """Admissions, chunks, decode steps with padded entries and releases, in any order."""
    rng = random.Random(seed)
    reqs, width = rng.choice([(3, 200), (17, 1000), (70, 700)])
    blocks = 1 + reqs * -(-width // 64)
    pool, want = BlockReqToTokenPool(reqs, width, blocks, cuda), of.Slots(reqs, width, blocks)
    lens = [0] * reqs
    for _ in range(30):
        some = rng.sample(range(reqs), rng.randint(1, reqs))
        act = rng.random()
        if act < 0.4:
            new = [rng.choice([0, 1, rng.randint(0, width - lens[r])]) if lens[r] < width else 0 for r in some]
            total = sum(new) + rng.choice([0, 0, 5])
            loc, pos = want.assign(some, [lens[r] for r in some], new, total)
            got = pool.assign(i64(some, cuda), i64([lens[r] for r in some], cuda), i64(new, cuda), total)
            for r, n in zip(some, new):
                lens[r] += n
        elif act < 0.8:
            seq = [lens[r] + 1 if lens[r] < width and rng.random() < 0.8 else 0 for r in some]
            parts = [want.assign([r], [s - 1], [1], 1) if s else (np.zeros(1, int),) * 2 for r, s in zip(some, seq)]
            loc, pos = (np.concatenate([p[i] for p in parts]) for i in range(2))
            got = pool.assign_decode(i64(some, cuda), i64(seq, cuda))
            for r, s in zip(some, seq):
                lens[r] = max(lens[r], s)
        else:
            some = some[: max(1, reqs // 2)]
            want.release(some)
            pool.release(i64(some, cuda))
            loc = pos = got = None
            for r in some:
                lens[r] = 0
        check(pool, want, loc, pos, got)
    pool.check_errors()
    assert pool.available_blocks() == len(want.stack)


@pytest.mark.parametrize("reqs", [1, 1025, 2500])
def test_more_requests_than_the_plan_s_threads(cuda, reqs):
    rng = random.Random(reqs)
    width = 130
    pool, want = BlockReqToTokenPool(reqs, width, 1 + 3 * reqs, cuda), of.Slots(reqs, width, 1 + 3 * reqs)
    order = rng.sample(range(reqs), reqs)
    new = [rng.randint(0, 100) for _ in order]
    loc, pos = want.assign(order, [0] * reqs, new, sum(new))
    got = pool.assign(i64(order, cuda), i64([0] * reqs, cuda), i64(new, cuda), sum(new))
    check(pool, want, loc, pos, got)
    held = {r: n for r, n in zip(order, new)}
    parts = [want.assign([r], [held[r]], [1], 1) for r in range(reqs)]
    got = pool.assign_decode(torch.arange(reqs), i64([held[r] + 1 for r in range(reqs)], cuda))
    check(pool, want, *(np.concatenate([p[i] for p in parts]) for i in range(2)), got)
    pool.release(i64(order, cuda))
    want.release(order)
    check(pool, want)


def test_asked_again_it_answers_the_same(cuda):
    pool = BlockReqToTokenPool(2, 500, 20, cuda)
    args = (i64([1, 0], cuda), i64([0, 0], cuda), i64([130, 64], cuda), 194)
    first = pool.assign(*args)
    free = pool.available_blocks()
    again = pool.assign(*args)
    assert all(torch.equal(a, b) for a, b in zip(first, again)) and pool.available_blocks() == free == 20 - 1 - 4


def test_a_prefix_that_was_skipped_has_its_blocks_too(cuda):
    """Tokens from position 200 on: the blocks of the 200 before them are handed out as well."""
    pool = BlockReqToTokenPool(2, 500, 20, cuda)
    loc, pos = pool.assign(i64([1], cuda), i64([200], cuda), i64([3], cuda), 3)
    assert pool.held.tolist() == [0, 4] and (pool.block_table[1, :4] > 0).all()
    assert pos.tolist() == [200, 201, 202] and loc.tolist() == [int(pool.block_table[1, 3]) * 64 + p % 64 for p in pos.tolist()]
    loc, pos = pool.assign_decode(i64([0], cuda), i64([130], cuda))
    assert pool.held.tolist() == [3, 4] and loc.tolist() == [int(pool.block_table[0, 2]) * 64 + 1]


def state(pool):
    return [t.clone() for t in (pool.block_table, pool.held, pool.free_blocks, pool.free_count, pool.req_to_token)]


@pytest.mark.parametrize("rpi, prefix, new, total, error", [
    ([0, 1], [0, 0], [300, 300], 600, RuntimeError),          # 10 blocks of 9
    ([0, 0], [0, 0], [10, 10], 20, ValueError),               # a request twice
    ([0, 2], [0, 0], [10, 10], 20, ValueError),               # a request outside the table
    ([0, -1], [0, 0], [10, 10], 20, ValueError),
    ([0, 1], [0, 495], [10, 10], 20, ValueError),             # past the table's width
    ([0, 1], [0, -1], [10, 10], 20, ValueError),
    ([0, 1], [0, 0], [10, -1], 20, ValueError),
    ([0, 1], [0, 0], [1 << 40, 10], 20, ValueError),
    ([0, 1], [0, 0], [10, 11], 20, ValueError),               # more tokens than announced
])
def test_a_refused_batch_takes_nothing(cuda, rpi, prefix, new, total, error):
    pool = BlockReqToTokenPool(2, 500, 10, cuda)
    pool.assign(i64([1], cuda), i64([0], cuda), i64([5], cuda), 5)
    before = state(pool)
    loc, pos = pool.assign(i64(rpi, cuda), i64(prefix, cuda), i64(new, cuda), total)
    assert not loc.any() and not pos.any()
    assert all(torch.equal(a, b) for a, b in zip(before, state(pool)))
    torch.cuda.synchronize()
    with pytest.raises(error):
        pool.poll_errors()
    pool.check_errors()  # raised once
    loc, _ = pool.assign(i64([0], cuda), i64([0], cuda), i64([500], cuda), 500)  # goes on
    assert (loc > 0).all()
    pool.check_errors()


@pytest.mark.parametrize("poll", [True, False])
def test_a_refusal_behind_another_is_raised_as_well(cuda, poll):
    """A call that is refused while an earlier refusal is looked at: each of them is raised, once,
    whether its kernel had run by then or not."""
    pool = BlockReqToTokenPool(2, 500, 10, cuda)
    work = torch.randn(4096, 4096, device=cuda)
    for _ in range(3):
        said = []
        pool.assign(i64([0, 1], cuda), i64([0, 0], cuda), i64([300, 300], cuda), 600)  # 10 blocks of 9
        torch.cuda.synchronize()
        twice = i64([0, 0], cuda), i64([0, 0], cuda), i64([10, 10], cuda)
        for _ in range(20):
            work = work @ work * 1e-2
        pool.assign(*twice, 20)
        for check in (pool.poll_errors if poll else pool.check_errors, pool.check_errors):
            try:
                check()
            except (RuntimeError, ValueError) as e:
                said.append(str(e))
        assert sum("out of memory" in s for s in said) == 1 and sum("twice" in s for s in said) == 1, said
        torch.cuda.synchronize()
        pool.poll_errors()
        pool.check_errors()


def test_a_call_refused_for_two_reasons(cuda):
    pool = BlockReqToTokenPool(2, 500, 3, cuda)
    pool.assign(i64([0, 0], cuda), i64([0, 0], cuda), i64([300, 300], cuda), 500)
    with pytest.raises(ValueError, match="out of memory.*twice.*total"):
        pool.check_errors()
    torch.cuda.synchronize()
    pool.poll_errors()


def test_refused_decode_and_release(cuda):
    pool = BlockReqToTokenPool(3, 200, 3, cuda)
    loc, pos = pool.assign_decode(i64([0, 1, 2], cuda), i64([1, 1, 1], cuda))  # 3 blocks of 2
    assert not loc.any() and not pos.any()
    with pytest.raises(RuntimeError, match="out of memory"):
        pool.check_errors()
    pool.assign_decode(i64([0, 0, 1], cuda), i64([1, 0, 1], cuda))  # padding may name anyone
    pool.check_errors()
    before = state(pool)
    for bad in ([0, 0], [0, 3], [-1]):
        pool.release(i64(bad, cuda))
        assert all(torch.equal(a, b) for a, b in zip(before, state(pool)))
        with pytest.raises(ValueError):
            pool.check_errors()
    pool.release(i64([], cuda))
    assert pool.assign(i64([], cuda), i64([], cuda), i64([], cuda), 0)[0].numel() == 0
    assert pool.assign(i64([2], cuda), i64([0], cuda), i64([0], cuda), 4)[0].tolist() == [0] * 4
    pool.check_errors()


def test_arguments_are_checked(cuda):
    pool = BlockReqToTokenPool(2, 500, 10, cuda)
    one, two = i64([0], cuda), i64([0, 1], cuda)
    with pytest.raises(ValueError, match="length"):
        pool.assign(one, two, one, 3)
    with pytest.raises(ValueError, match="length"):
        pool.assign_decode(one, two)
    with pytest.raises(ValueError, match="one-dimensional"):
        pool.assign_decode(two.view(1, 2), two)
    with pytest.raises(ValueError, match="whole"):
        pool.assign_decode(two, two.float())
    with pytest.raises(ValueError, match="total"):
        pool.assign(one, one, one, -1)
    for bad in ((2, 500, 0), (2, 500, (1 << 24) + 1), (0, 500, 4), ((1 << 18) + 1, 1, 4), (2, 0, 4), (2, 1 << 30, 4)):
        with pytest.raises(ValueError):
            BlockReqToTokenPool(*bad, cuda)


def test_slots_and_blocks_come_back_together(cuda):
    pool = BlockReqToTokenPool(2, 500, 10, cuda)
    r = pool.alloc()
    pool.assign(i64([r], cuda), i64([0], cuda), i64([100], cuda), 100)
    assert pool.available_size() == 1 and pool.available_blocks() == 7
    pool.free(r)
    assert pool.available_size() == 2 and pool.available_blocks() == 9 and not pool.req_to_token.any()


def test_decode_slots_in_a_replayed_graph(cuda):
    """A captured step replayed while the lengths grow in place, eager calls between the replays."""
    pool, want = BlockReqToTokenPool(4, 400, 40, cuda), of.Slots(4, 400, 40)
    rpi, seq = i64([2, 0, 3], cuda), i64([61, 0, 128], cuda)
    pool.assign_decode(rpi, seq)
    for r, s in ((2, 61), (3, 128)):
        want.assign([r], [s - 1], [1], 1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loc, pos = pool.assign_decode(rpi, seq)
    for step in range(9):
        seq[0] += 1
        seq[2] += 1
        if step == 4:
            pool.assign(i64([1], cuda), i64([0], cuda), i64([70], cuda), 70)
            want.assign([1], [0], [70], 70)
        graph.replay()
        parts = [want.assign([r], [s - 1], [1], 1) if s else (np.zeros(1, int),) * 2
                 for r, s in zip([2, 0, 3], seq.tolist())]
        check(pool, want, *(np.concatenate([p[i] for p in parts]) for i in range(2)), (loc, pos))
    pool.check_errors()


def test_a_prompt_s_slots_in_a_replayed_graph(cuda):
    pool = BlockReqToTokenPool(3, 3000, 200, cuda)
    rpi, prefix, new = i64([2, 1], cuda), i64([0, 0], cuda), i64([900, 1100], cuda)
    graph = torch.cuda.CUDAGraph()
    pool.assign(rpi, prefix, new, 2000)
    pool.release(rpi)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        loc, pos = pool.assign(rpi, prefix, new, 2000)
        pool.release(rpi)
    fresh = pool.free_blocks.clone()
    for a, b in ((900, 1100), (1, 64), (1000, 0)):
        new.copy_(i64([a, b], cuda))
        graph.replay()
        want = of.Slots(3, 3000, 200).assign([2, 1], [0, 0], [a, b], 2000)
        assert np.array_equal(loc.cpu().numpy(), want[0]) and np.array_equal(pos.cpu().numpy(), want[1])
        assert torch.equal(pool.free_blocks, fresh) and pool.available_blocks() == 199 and not pool.block_table.any()
    pool.check_errors()


def test_another_stream(cuda):
    pool = BlockReqToTokenPool(2, 5000, 100, cuda)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        loc, pos = pool.assign(i64([0], cuda), i64([0], cuda), i64([4000], cuda), 4000)
    s.synchronize()
    want = of.Slots(2, 5000, 100).assign([0], [0], [4000], 4000)
    assert np.array_equal(loc.cpu().numpy(), want[0]) and np.array_equal(pos.cpu().numpy(), want[1])
