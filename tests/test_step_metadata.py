"""nvk_step_metadata and nvk_release_blocks against a plain restatement (ref_blocks8.py): whole numbers, so equal to the last one."""
import ctypes
import itertools

import numpy as np
import pytest

import ref_blocks8 as ref
from util import entry, nvk


@pytest.fixture(scope="module")
def built():
    entry.build()
    return nvk()


# ---- on the CPU --------------------------------------------------------------------------------------------------------------
def test_by_hand():
    # Blocks of 4: a request of 5 tokens grows by 4 to 9 (3 blocks, one of them new), one of 4 by 1 (2 blocks), one of 8 by none.
    r = ref.Requests([5, 4, 8], [[1, 2, -1], [3, -1, -1], [4, 5, -1]], [7, 8, 9], 3, 4)
    tables, ctx, cu_q, cu_k, positions, slots = r.step([4, 1, 0], None, 3, 6, 10)
    assert tables == [[1, 2, 9], [3, 8, 0], [4, 5, 0]] and ctx == [9, 5, 8] and cu_q == [0, 4, 5, 5] and cu_k == [0, 9, 14, 22]
    assert positions == [5, 6, 7, 8, 4, 0] and slots == [9, 10, 11, 36, 32, -1] and r.count == 1 and r.lens == [9, 5, 8]
    # One free block: the first of two that need one gets it, the third needs none.
    r = ref.Requests([4, 4, 5], [[1, -1], [2, -1], [3, 4]], [5], 1, 4)
    assert r.step([1, 1, 1], None, 2, 3, 6)[:2] == ([[1, 5], [0, 0], [3, 4]], [5, 0, 6]) and r.count == 0 and r.lens == [5, 4, 6]
    r.release([2, 0], [1, 0])
    assert r.lens == [0, 4, 0] and r.free == [4] and r.count == 1   # (no room for the others)


L, I = ctypes.c_int64, ctypes.c_int
P, ODD = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 2)
AT = [ctypes.c_void_p(i << 40) for i in range(1, 16)]       # (nothing is read there)
LENS, COUNT, BLOCKS, FREE, NEW, TABLES = AT[0], AT[1], AT[2], AT[3], AT[4], AT[5]


def _step_args(**change):
    a = dict(new=NEW, rows=None, lens=LENS, blocks=BLOCKS, free=FREE, count=COUNT, batch=L(2), num_rows=L(4), row_blocks=L(8), num_free=L(16), cache=L(64), bs=I(16),
             tables=TABLES, width=L(8), ctx=AT[6], cu_q=AT[7], cu_k=AT[8], pos=AT[9], slots=AT[10], tokens=L(8), new_lens=LENS, new_count=COUNT, dtype=I(3), stream=None)
    a.update(change)
    return a.values()


def _release_args(**change):
    a = dict(rows=P, first=None, lens=LENS, blocks=BLOCKS, free=FREE, count=COUNT, batch=L(2), num_rows=L(4), row_blocks=L(8), num_free=L(16), bs=I(16), new_lens=LENS,
             new_count=COUNT, dtype=I(3), stream=None)
    a.update(change)
    return a.values()


def _call(lib, name, *args):
    rc = getattr(lib.lib(), name)(*args)
    return rc, lib.lib().nvk_last_error().decode()


@pytest.mark.parametrize("change,code,word", [
    (dict(new=None), 1, "defined"), (dict(lens=None), 1, "defined"), (dict(tables=None), 1, "defined"), (dict(new_count=None), 1, "defined"),
    (dict(pos=None), 1, "defined"), (dict(dtype=I(1)), 1, "int32 or int64"), (dict(batch=L(-1)), 1, "positive"), (dict(bs=I(0)), 1, "positive"),
    (dict(width=L(0)), 1, "positive"), (dict(tokens=L(-1)), 1, "positive"), (dict(batch=L(5)), 1, "row for every request"), (dict(new=ODD), 1, "misaligned"),
    (dict(lens=ODD), 1, "misaligned"), (dict(dtype=I(4), new_lens=ctypes.c_void_p(LENS.value + 8)), 1, "overlap"), (dict(new_lens=ctypes.c_void_p(LENS.value + 4)), 1, "overlap"),
    (dict(ctx=LENS), 1, "overlaps"), (dict(ctx=NEW), 1, "overlaps"), (dict(tables=BLOCKS), 1, "overlaps"), (dict(pos=AT[10]), 1, "overlaps"), (dict(rows=P, cu_q=P), 1, "overlaps"),
    (dict(new_count=FREE), 1, "overlaps"), (dict(new_lens=COUNT), 1, "overlaps"), (dict(slots=FREE), 1, "overlaps"), (dict(width=L(1 << 45)), 3, "too many"),
    (dict(row_blocks=L(1 << 45)), 3, "too many"), (dict(tokens=L(1 << 45)), 3, "too many"),
    (dict(cache=L(1 << 28)), 1, "int64"), (dict(rows=P, batch=L(8193)), 3, "at most 8192"), (dict(rows=P, batch=L(8192), width=L(1 << 20)), 3, "too many"),
    (dict(batch=L(0)), 1, "positive")])
def test_step_refuses(built, change, code, word):
    rc, said = _call(built, "nvk_step_metadata", *_step_args(**change))
    assert rc == code and (rc == 0 or word in said), said


@pytest.mark.parametrize("change,code,word", [
    (dict(lens=None), 1, "defined"), (dict(free=None), 1, "defined"), (dict(dtype=I(0)), 1, "int32 or int64"), (dict(num_rows=L(0)), 1, "positive"),
    (dict(rows=None, batch=L(5)), 1, "row for every request"), (dict(first=ODD), 1, "misaligned"), (dict(new_lens=ctypes.c_void_p(LENS.value + 4)), 1, "overlap"),
    (dict(free=BLOCKS), 1, "overlaps"), (dict(rows=P, free=P), 1, "overlaps"), (dict(new_count=FREE), 1, "overlaps"), (dict(row_blocks=L(1 << 45)), 3, "too many"),
    (dict(rows=P, batch=L(9000)), 3, "at most 8192"), (dict(batch=L(-1)), 1, "positive")])
def test_release_refuses(built, change, code, word):
    rc, said = _call(built, "nvk_release_blocks", *_release_args(**change))
    assert rc == code and (rc == 0 or word in said), said


# ---- on the GPU --------------------------------------------------------------------------------------------------------------
class Tables:
    """The same tables here and on the GPU."""

    def __init__(self, rng, rows, row_blocks, block_size, spare, longest=None, dtype="int32"):
        import torch
        self.torch, self.dtype, self.bs = torch, getattr(torch, dtype), block_size
        lens = rng.integers(0, (longest if longest is not None else row_blocks * block_size) + 1, rows)
        need = -(-lens // block_size)
        perm = rng.permutation(int(need.sum()) + spare)
        held, at = np.full((rows, row_blocks), -7, np.int64), 0
        for i, n in enumerate(need):
            held[i, :n] = perm[at:at + n]
            at += n
        free = np.full(len(perm), -9, np.int64)
        free[:spare] = perm[at:]
        self.pool = len(perm)
        self.ref = ref.Requests(lens.tolist(), held.tolist(), free.tolist(), spare, block_size)
        self.lens, self.held, self.free, self.count = (self.up(v) for v in (lens, held, free, [spare]))

    def up(self, v):
        return self.torch.as_tensor(np.asarray(v), dtype=self.dtype).cuda()

    def step(self, new, rows, width, tokens, apart=False, sums=True):
        t = self.torch
        full = lambda *shape: t.full(shape, -99, dtype=self.dtype, device="cuda")
        b = len(new)
        out = [full(b, width), full(b), full(b + 1) if sums else None, full(b + 1) if sums else None, full(tokens), full(tokens)]
        # apart: True, or "lens" or "count": only those have a tensor of their own to go to
        to = t.full_like(self.lens, -99) if apart in (True, "lens") else None, t.full_like(self.count, -99) if apart in (True, "count") else None
        before = self.lens.clone(), self.count.clone()
        nvk().step_metadata(self.up(new), None if rows is None else self.up(rows), self.lens, self.held, self.free, self.count, self.bs, self.pool, *out, *to)
        want = self.ref.step(new, rows, width, tokens, self.pool)
        if to[0] is not None:
            assert t.equal(before[0], self.lens)
            self.lens = to[0]
        if to[1] is not None:
            assert t.equal(before[1], self.count)
            self.count = to[1]
        for name, got, w in zip(("tables", "ctx", "cu_q", "cu_k", "positions", "slots"), out, want):
            assert got is None or got.tolist() == w, name
        self.same()
        return out

    def release(self, rows, first, apart=False):
        t = self.torch
        to = (t.full_like(self.lens, -99), t.full_like(self.count, -99)) if apart else (None, None)
        nvk().release_blocks(None if rows is None else self.up(rows), None if first is None else self.up(first), self.lens, self.held, self.free, self.count,
                             self.bs, *to)
        self.ref.release(rows, first)
        if apart:
            self.lens, self.count = to
        self.same()

    def same(self):
        assert self.lens.tolist() == self.ref.lens and self.count.tolist() == [self.ref.count]
        assert self.held.tolist() == self.ref.held and self.free.tolist() == self.ref.free


@pytest.mark.gpu
@pytest.mark.parametrize("batch,dtype,apart", [(1, "int32", False), (3, "int64", True), (33, "int32", True), (511, "int64", False), (513, "int32", False),
                                               (1024, "int32", True), (1700, "int64", False)])
@pytest.mark.parametrize("block_size,row_blocks", [(1, 9), (16, 5), (256, 3), (24, 40)])
def test_steps_one_after_the_other(batch, dtype, apart, block_size, row_blocks):
    rng = np.random.default_rng(batch * 1000 + block_size)
    t = Tables(rng, batch + 5, row_blocks, block_size, 2 * batch, dtype=dtype)
    for n in range(3):
        rows = rng.permutation(batch + 5)[:batch]
        rows[rng.random(batch) < 0.05] = rng.choice([-1, batch + 5, 1 << 30])             # padding
        new = rng.integers(0, 3, batch) * rng.integers(0, 2 + block_size // 2, batch)
        total = int(new.sum())
        t.step(new.tolist(), rows.tolist(), rng.choice([row_blocks, max(1, row_blocks - 1), row_blocks + 2]), max(0, total + (5, 0, -3)[n]), apart)
        done = rng.permutation(batch + 5)[:batch // 4]
        t.release(done.tolist(), None if n == 0 else rng.integers(0, row_blocks + 1, len(done)).tolist(), apart)


@pytest.mark.gpu
def test_decode_steps_until_the_blocks_are_gone_and_back():
    rng = np.random.default_rng(3)
    t = Tables(rng, 40, 6, 16, 30, longest=40)
    stalled = 0
    for _ in range(40):
        out = t.step([1] * 40, None, 6, 40, sums=False)
        stalled += out[1].tolist().count(0)
    assert stalled > 0
    t.release(None, None)
    assert t.count.item() == t.pool
    t.step([1] * 40, None, 6, 48)


@pytest.mark.gpu
def test_a_shortage_is_the_same_for_all_that_come_after_it_but_those_that_need_nothing():
    rng = np.random.default_rng(4)
    t = Tables(rng, 8, 4, 16, 3, longest=0)
    for i, n in enumerate((16, 5, 0, 31, 64, 0, 16, 1)):
        t.ref.lens[i] = n
    used = itertools.count(100)
    t.ref.held = [[next(used) if j < -(-n // 16) else -7 for j in range(4)] for n in t.ref.lens]
    t.lens, t.held = t.up(t.ref.lens), t.up(t.ref.held)
    out = t.step([1, 11, 33, 1, 1, 0, 40, 3], None, 4, 100)    # 1 block, 0, 3 (no), 0, too long, nothing, 3 (no), 0
    assert out[1].tolist() == [17, 16, 0, 32, 0, 0, 0, 4]
    assert out[4].tolist()[12:45] == [0] * 33 and out[5].tolist()[12:45] == [-1] * 33


@pytest.mark.gpu
def test_lengths_and_ids_out_of_range():
    import torch
    t = Tables(np.random.default_rng(5), 4, 3, 16, 6, longest=30)
    # what no program should hand over: lengths and counts out of range; they are kept to the tables' sizes
    lens = torch.tensor([-5, 2 ** 31 - 1, 100, 20], dtype=torch.int32, device="cuda")
    count = torch.tensor([1000], dtype=torch.int32, device="cuda")
    new = torch.tensor([3, 5, -1, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    tables, ctx = torch.full((4, 3), -9, dtype=torch.int32, device="cuda"), torch.full((4,), -9, dtype=torch.int32, device="cuda")
    cu = torch.full((5,), -9, dtype=torch.int32, device="cuda")
    positions, slots = (torch.full((12,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    nvk().step_metadata(new, None, lens, t.held, t.free, count, 16, t.pool, tables, ctx, cu, None, positions, slots)
    assert ctx.tolist() == [3, 0, 0, 0] and count.tolist() == [t.pool - 1] and cu.tolist() == [0, 3, 8, 8, 2 ** 31 - 1]
    assert positions.tolist()[:3] == [0, 1, 2] and slots.tolist()[3:] == [-1] * 9


@pytest.mark.gpu
def test_blocks_outside_the_cache_give_no_slots():
    t = Tables(np.random.default_rng(6), 2, 3, 16, 6, longest=0)
    t.ref.free[5] = t.pool + 3
    t.free = t.up(t.ref.free)
    out = t.step([4, 4], None, 3, 8)
    assert out[5].tolist()[:4] == [-1] * 4 and min(out[5].tolist()[4:]) >= 0


@pytest.mark.gpu
@pytest.mark.parametrize("batch,width,tokens", [(8192, 7, 20000), (64, 2048, 70000), (1100, 128, 300000), (8192, 64, 9000), (8192, 2, 5000)])
@pytest.mark.parametrize("dtype,apart", [("int64", False), ("int32", True), ("int32", False)])
def test_the_largest_batch_and_wide_tables(batch, width, tokens, dtype, apart):
    """Steps of many blocks, twice in a row (what is updated in place follows in a kernel of its own)."""
    rng = np.random.default_rng(7)
    t = Tables(rng, batch + 1, width, 4, batch * 2, dtype=dtype)
    for _ in range(2):
        new = rng.integers(0, 4, batch) if batch > 100 else rng.integers(0, 2000, batch)
        t.step(new.tolist(), (rng.permutation(batch + 1)[:batch]).tolist(), width, tokens, apart)
    t.release(rng.permutation(batch + 1)[:batch].tolist(), None, apart)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,width,tokens", [(7, 9, 30), (250, 40, 600), (90, 2000, 400), (1000, 12, 3000), (1500, 300, 5000)])
@pytest.mark.parametrize("dtype", ["int64", "int32"])
@pytest.mark.parametrize("apart", ["lens", "count"])
def test_only_lengths_or_only_the_count_in_place(batch, width, tokens, dtype, apart):
    """In one cluster and by many blocks; with blocks for all, then for a few."""
    rng = np.random.default_rng(batch)
    t = Tables(rng, batch + 2, width, 4, batch * 2, dtype=dtype)
    for _ in range(3):
        t.step(rng.integers(0, 4, batch).tolist(), rng.permutation(batch + 2)[:batch].tolist(), width, tokens, apart)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,width", [(5, 8), (300, 16), (2000, 96)])
def test_tables_and_tokens_at_odd_addresses(batch, width):
    """Tables, positions and slots that begin off a 16-byte boundary; counts of tokens that are no multiple of four."""
    import torch
    rng = np.random.default_rng(batch)
    t = Tables(rng, batch, width, 16, batch * 2, dtype="int32")
    odd = lambda *shape: torch.full((1 + int(np.prod(shape)),), -99, dtype=torch.int32, device="cuda")[1:].view(shape)
    new = rng.integers(0, 40, batch).tolist()
    tokens = sum(new) + 1
    held = odd(batch, width)
    held.copy_(t.held)
    out = [odd(batch, width), odd(batch), odd(batch + 1), odd(batch + 1), odd(tokens), odd(tokens)]
    nvk().step_metadata(t.up(new), None, t.lens, held, t.free, t.count, 16, t.pool, *out)
    want = t.ref.step(new, None, width, tokens, t.pool)
    assert [o.tolist() for o in out] == list(want)
    assert held.tolist() == t.ref.held and t.lens.tolist() == t.ref.lens and t.count.tolist() == [t.ref.count]


@pytest.mark.gpu
def test_two_steps_at_once_on_two_streams():
    """Two sets of tables, one step each, at the same time: nothing is shared between calls."""
    import torch
    rng = np.random.default_rng(12)
    sets = [Tables(rng, 200, 40, 16, 300, dtype="int32") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in sets]
    new = [rng.integers(0, 30, 200).tolist() for _ in sets]
    outs = []
    for t, n in zip(sets, new):
        full = lambda *shape: torch.full(shape, -99, dtype=torch.int32, device="cuda")
        outs.append((t.up(n), [full(200, 40), full(200), full(201), full(201), full(sum(n)), full(sum(n))]))
    torch.cuda.synchronize()
    for t, st, (n, out) in zip(sets, streams, outs):
        with torch.cuda.stream(st):
            nvk().step_metadata(n, None, t.lens, t.held, t.free, t.count, 16, t.pool, *out)
    torch.cuda.synchronize()
    for t, n, (_, out) in zip(sets, new, outs):
        assert [o.tolist() for o in out] == list(t.ref.step(n, None, 40, sum(n), t.pool))
        t.same()


@pytest.mark.gpu
def test_captured_steps_go_on_from_one_another():
    """A decode loop as a CUDA graph: lengths, blocks and the count move on with every replay."""
    import torch
    t = Tables(np.random.default_rng(8), 6, 4, 16, 20, longest=20)
    new = t.up([1] * 6)
    full = lambda *shape: torch.full(shape, -99, dtype=t.dtype, device="cuda")
    out = [full(6, 4), full(6), full(7), full(7), full(8), full(8)]
    stream = torch.cuda.Stream()
    lens, held, count = t.lens.clone(), t.held.clone(), t.count.clone()
    with torch.cuda.stream(stream):
        nvk().step_metadata(new, None, t.lens, t.held, t.free, t.count, 16, t.pool, *out)   # (warm-up, undone)
    stream.synchronize()
    t.lens.copy_(lens); t.held.copy_(held); t.count.copy_(count)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        nvk().step_metadata(new, None, t.lens, t.held, t.free, t.count, 16, t.pool, *out)
    for _ in range(30):
        graph.replay()
        want = t.ref.step([1] * 6, None, 4, 8, t.pool)
        torch.cuda.synchronize()
        assert [o.tolist() for o in out] == list(want)
        t.same()


@pytest.mark.gpu
@pytest.mark.parametrize("change,word", [
    (dict(new="int64"), "dtype of the other"), (dict(lens="float32"), "int32 or int64"), (dict(tables=(3, 4)), "row for every element"),
    (dict(cu=(4,)), "one element more"), (dict(slots=(7,)), "same size"), (dict(count=(2,)), "one element"), (dict(held=(5, 4)), "row, new_request_lens"),
    (dict(free="cpu"), "CUDA")])
def test_the_binding_refuses(change, word):
    import torch
    shapes = dict(new=(4,), lens=(4,), held=(4, 4), free=(9,), count=(1,), tables=(4, 4), ctx=(4,), cu=(5,), pos=(8,), slots=(8,))
    kind, device = dict.fromkeys(shapes, torch.int32), dict.fromkeys(shapes, "cuda")
    for name, v in change.items():
        if v == "cpu":
            device[name] = v
        elif isinstance(v, str):
            kind[name] = getattr(torch, v)
        else:
            shapes[name] = v
    x = {n: torch.zeros(shapes[n], dtype=kind[n], device=device[n]) for n in shapes}
    with pytest.raises(ValueError, match=word):
        nvk().step_metadata(x["new"], None, x["lens"], x["held"], x["free"], x["count"], 16, 64, x["tables"], x["ctx"], x["cu"], None, x["pos"], x["slots"])


# ---- the barrier of the cluster ------------------------------------------------------------------------------------------------
def test_no_barrier_asks_a_warp_to_come_together():
    """The .aligned forms of the cluster's barrier are undefined where a warp's threads come from loops and branches of their own, as here."""
    import os
    import re
    source = open(os.path.join(os.path.dirname(entry.__file__), "nano-vllm-cpp_b200", "csrc", "step_metadata.cu")).read()
    forms = re.findall(r"barrier\.cluster\.(?:arrive|wait)[a-z.]*", source)
    assert len(forms) >= 2 and not any("aligned" in f for f in forms), forms


@pytest.mark.gpu
@pytest.mark.parametrize("apart", [False, "lens", "count"])
@pytest.mark.parametrize("batch,rows,width,dtype", [(37, 1003, 13, "int32"), (255, 300, 37, "int64"), (700, 1301, 9, "int32")])
def test_clusters_with_ragged_work(batch, rows, width, dtype, apart):
    """Requests, table entries, tokens and rows that leave warps with threads of unequal work before the barrier; steps and releases in turn, in place."""
    rng = np.random.default_rng(batch)
    t = Tables(rng, rows, width, 8, 3 * batch, longest=5 * 8, dtype=dtype)
    for n in range(12):
        mine = rng.permutation(rows)[:batch]
        mine[rng.random(batch) < 0.1] = -1
        new = rng.integers(0, 9, batch) * (rng.random(batch) < 0.7)
        t.step(new.tolist(), mine.tolist(), width, int(new.sum()) + n, apart)
        done = rng.permutation(rows)[:int(rng.integers(1, batch))]
        t.release(done.tolist(), rng.integers(0, 3, len(done)).tolist() if n % 2 else None)


def test_reads_of_the_other_blocks_come_before_the_first_ones_writes():
    """Lengths and count are written in place behind a barrier: whoever reads them has to arrive with release, and the writer to wait with acquire."""
    import os
    import re
    source = open(os.path.join(os.path.dirname(entry.__file__), "nano-vllm-cpp_b200", "csrc", "step_metadata.cu")).read()
    assert re.search(r"if \(first_block\) asm[^;]*barrier\.cluster\.arrive\.relaxed;[^;]*;\s*else asm[^;]*barrier\.cluster\.arrive\.release;", source)
    assert "barrier.cluster.wait.acquire;" in source


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["int32", "int64"])
@pytest.mark.parametrize("batch,width", [(9, 100), (60, 300), (300, 700)])
def test_many_releases_in_place(batch, width, dtype):
    """The count and the lengths written by one block of a cluster while the others still work: the same tables over and over, by clusters of 2 to 16 blocks."""
    import torch
    rng = np.random.default_rng(width)
    t = Tables(rng, batch + 3, width, 2, 50, dtype=dtype)
    done = rng.permutation(batch + 3)[:batch]
    rows, first = t.up(done), t.up(rng.integers(0, 3, batch))
    lens, free, count = t.lens.clone(), t.free.clone(), t.count.clone()
    t.ref.release(done.tolist(), first.tolist())
    want = t.up(t.ref.lens), t.up(t.ref.free), t.up([t.ref.count])
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(300):
        t.lens.copy_(lens); t.free.copy_(free); t.count.copy_(count)
        nvk().release_blocks(rows, first, t.lens, t.held, t.free, t.count, 2)
        for got, w in zip((t.lens, t.free, t.count), want):
            wrong += (got != w).sum()
    assert wrong.item() == 0
    t.same()
