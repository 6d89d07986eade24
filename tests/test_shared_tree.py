"""The node-local shared-host tree pool (parallel/shared_tree.py): every rank
makes the same slot choice from the gathered free masks, a slot a rank still
views is never reused, and ranks of one machine see each other's writes after
the flag barrier. Host memory stands in for the HIP registration (no GPU)."""
import multiprocessing as mp

import numpy as np
import pytest

from mpitree_amd.parallel import shared_tree as st


class _FakeHip:
    def host_register(self, p, n):
        return p  # (the device pointer of a mapped host range)

    def host_unregister(self, p):
        pass


class _Comm:
    def __init__(self, rank, P):
        self.rank, self.world_size = rank, P


def _pool(rank=0, P=2, uid=None):
    return st.ShmTreePool(_Comm(rank, P), _FakeHip(), uid if uid is not None else 0x5EED + rank)


def test_choose_reuses_only_slots_free_everywhere():
    pool = _pool()
    a = pool.choose([0, 0], 1000)  # nothing exists: a new slot
    assert a.nbytes - st.HEADER >= 1000 and pool.free_mask() == 1
    view = a.nd[st.HEADER : st.HEADER + 64]  # a tree this rank still holds
    assert pool.free_mask() == 0
    b = pool.choose([pool.free_mask(), 1], 1000)  # busy here: another slot
    assert b is not a
    del view
    assert pool.free_mask() == 3
    # the peer still holds slot 0: slot 1 is the only one free everywhere
    assert pool.choose([3, 2], 1000) is b
    # too small everywhere: a new, larger slot
    c = pool.choose([3, 3], 10 << 20)
    assert c is not a and c is not b and c.nbytes - st.HEADER >= 10 << 20
    for sl in list(pool.slots.values()):
        sl.close()


def test_next_slot_is_agreed_ahead_and_excludes_the_current():
    pool = _pool()
    cur = pool.choose([0, 0], 4096)
    pool.plan_next([pool.free_mask(), pool.free_mask()], cur, 4096)
    nxt = pool.take_next()
    assert nxt is not None and nxt is not cur and pool.take_next() is None
    for sl in list(pool.slots.values()):
        sl.close()


def test_short_dev_shm_refuses_a_new_slot_but_reuses_one():
    pool = _pool()
    a = pool.choose([0, 0], 1 << 20)
    small = [st.SHM_MARGIN, 10 * st.SHM_MARGIN]  # one rank's /dev/shm is nearly full
    # a new slot would not fit beside the margin on that rank: every rank falls back
    assert pool.choose([0, 0], 1 << 20, shm_free=small) is None
    # an existing free slot costs no /dev/shm: it is still chosen
    assert pool.choose([1, 1], 1 << 20, shm_free=small) is a
    pool.plan_next([1, 1], a, 1 << 20, shm_free=small)
    assert pool.take_next() is None
    assert st.shm_free_bytes() >= 0
    for sl in list(pool.slots.values()):
        sl.close()


def _rank_main(rank, uid, q):
    pool = st.ShmTreePool(_Comm(rank, 2), _FakeHip(), uid)
    slot = pool.choose([0, 0], 1 << 16)  # same name on both ranks
    data = slot.nd[st.HEADER : st.HEADER + (1 << 16)].view(np.int64)
    half = data.size // 2
    data[rank * half : (rank + 1) * half] = rank + 1  # this rank's nodes
    pool.barrier(slot)
    q.put((rank, int(data[:half].sum()), int(data[half:].sum()), half))
    del data
    slot.close()


@pytest.mark.timeout(60)
def test_two_ranks_share_one_buffer_through_the_barrier():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    uid = int.from_bytes(np.random.default_rng().bytes(5), "little")
    ps = [ctx.Process(target=_rank_main, args=(r, uid, q)) for r in range(2)]
    for p in ps:
        p.start()
    got = sorted(q.get(timeout=50) for _ in range(2))
    for p in ps:
        p.join(20)
        assert p.exitcode == 0
    for rank, s0, s1, half in got:
        assert s0 == half and s1 == 2 * half  # both ranks' halves, seen by each


def test_pool_belongs_to_the_group_not_the_communicator():
    """Estimators build a communicator per fit: the pool (and its registered
    buffers) is found again through the process group, the host-key all-gather
    runs once."""
    calls = []

    class _G:  # a process group stand-in (weak-referenceable)
        pass

    class _C(_Comm):
        def _all_gather(self, a):
            calls.append(1)
            return np.stack([a, a])

    g = _G()
    a, b = _C(0, 2), _C(0, 2)
    a.group = b.group = g
    p1 = st.pool_for(a, _FakeHip())
    p2 = st.pool_for(b, _FakeHip())
    assert p1 is not None and p1 is p2 and len(calls) == 1
    c = _C(0, 2)
    c.group = _G()  # another group: another pool
    assert st.pool_for(c, _FakeHip()) is not p1 and len(calls) == 2


def test_exact_own_positions_group_jobs_by_owner():
    import torch

    from mpitree_amd.ops.exact_grower import _owners, own_positions

    # jobs {start, count, ...} in finisher order; owners dealt serpentine
    fj = torch.tensor([[0, 5, 0, 0, 0], [10, 3, 0, 0, 0], [20, 4, 0, 0, 0],
                       [30, 2, 0, 0, 0], [40, 1, 0, 0, 0]], dtype=torch.int64)
    own = _owners(5, 2, fj.device)
    pos, sizes = own_positions(fj, own, 2)
    want = {0: [], 1: []}
    for j in range(5):
        want[int(own[j])] += list(range(int(fj[j, 0]), int(fj[j, 0] + fj[j, 1])))
    assert sizes == [len(want[0]), len(want[1])]
    assert pos.tolist() == want[0] + want[1]


@pytest.mark.parametrize("C", [0, 2, 7])
@pytest.mark.parametrize("scattered", [False, True])
def test_two_ranks_nodes_make_one_tree(C, scattered):
    """Each rank copies the nodes its staging buffer holds (depth >= 0), whole runs of ids or
    scattered ones, and nothing else; together they are the tree."""
    N, width = 3000, 3 * 8 + 4 * C + 5 * 4
    assert sum(st._Slot.column_widths(width)) == width
    rng = np.random.default_rng(C)
    tree = rng.integers(0, 100, size=N * width, dtype=np.uint8)
    tree[-4 * N :].view(np.int32)[:] = rng.integers(0, 50, size=N)  # depths
    pool = _pool(uid=0x5EED00 + C + 100 * scattered)
    slot = pool.choose([0, 0], N * width)
    mine = rng.random(N) < 0.5 if scattered else (np.arange(N) // 700) % 2 == 0
    for own in (mine, ~mine):
        stage = rng.integers(0, 255, size=N * width, dtype=np.uint8)
        at = 0
        for w in st._Slot.column_widths(width):
            col = stage[at : at + N * w].reshape(N, w)
            col[own] = tree[at : at + N * w].reshape(N, w)[own]
            at += N * w
        stage[-4 * N :].view(np.int32)[~own] = -1
        slot.copy_nodes(stage, N)
    assert np.array_equal(slot.nd[st.HEADER : st.HEADER + N * width], tree)
    slot.close()


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("many", [False, True])
def test_runs_of_ids_make_one_tree(seed, many):
    """Segments in ascending order with prefix nodes between some of them, empty ones and
    neighbours: every id is written by one rank, and the copied nodes are the tree."""
    rng = np.random.default_rng(seed)
    P, S = 4, 900 if many else 30
    count = rng.integers(0, 4 if many else 60, size=S)
    gap = rng.integers(0, 3, size=S + 1) * (rng.random(S + 1) < 0.5)
    first = np.cumsum(gap[:-1]) + np.concatenate([[0], np.cumsum(count)[:-1]])
    N = int(gap.sum() + count.sum())
    segs = np.stack([first, count, rng.integers(0, P, size=S)], 1).astype(np.int64)
    segs = np.concatenate([segs, [[2 ** 63 - 1, 0, -1]]])  # (unused entries come last)
    owner = np.zeros(N, dtype=int)
    for a, c, r in segs[:-1].tolist():
        owner[a : a + c] = r
    C, width = 3, 3 * 8 + 4 * 3 + 5 * 4
    tree = rng.integers(0, 255, size=N * width, dtype=np.uint8)
    pool = _pool(uid=0x5EED500 + seed + 100 * many)
    slot = pool.choose([0, 0], N * width)
    for me in range(P):
        runs = st.own_runs(segs, N, me)
        mine = np.zeros(N, dtype=bool)
        for a, b in runs:
            assert a < b and not mine[a:b].any()
            mine[a:b] = True
        assert np.array_equal(mine, owner == me)
        assert all(b < a for (_, b), (a, _) in zip(runs, runs[1:]))  # (neighbours joined)
        stage, at = rng.integers(0, 255, size=N * width, dtype=np.uint8), 0
        for w in st._Slot.column_widths(width):
            part = slice(at, at + N * w)
            stage[part].reshape(N, w)[mine] = tree[part].reshape(N, w)[mine]
            at += N * w
        slot.copy_nodes(stage, N, runs)
    assert np.array_equal(slot.nd[st.HEADER : st.HEADER + N * width], tree)
    slot.close()
