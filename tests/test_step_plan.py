"""Page and slot bookkeeping of a step (plan_step, truncate, keep_rows): refusals on the CPU, and on the GPU every table,
slot, mask and moved byte against a plain restatement over Python lists."""
import ctypes
import random

import pytest
import torch

from phasorkv_b200 import PagedLatentCache, _lib, build

PAGE = 128


# ------------------------------------------------------------------------------------------------ restatement
class Tables:
    """Page tables, lengths and page stack as Python lists."""

    def __init__(self, table, lens, free):
        self.table, self.lens, self.free = table, lens, free

    def plan(self, new, cap, parents=None):
        """-> (cu, seq, positions, slots, mask) or None when the step is refused"""
        if any(m < 0 or L + m > len(self.table[0]) * PAGE for L, m in zip(self.lens, new)) or sum(new) > cap:
            return None
        need = [-(-(L + m) // PAGE) - -(-L // PAGE) for L, m in zip(self.lens, new)]
        if self.free is not None and sum(need) > len(self.free):
            return None
        cu, seq, pos, slots, mask = [0], [], [], [], []
        for b, (L, m) in enumerate(zip(self.lens, new)):
            if self.free is not None:
                for p in range(-(-L // PAGE), -(-(L + m) // PAGE)):
                    self.table[b][p] = self.free.pop()
            words, depth = [], []
            for i in range(m):
                t = L + i
                seq.append(b)
                slots.append(self.table[b][t // PAGE] * PAGE + t % PAGE)
                up = parents[cu[b] + i] if parents else i - 1
                depth.append(depth[up] + 1 if up >= 0 else 0)
                words.append((words[up] if up >= 0 else 0) | 1 << i)
                pos.append(L + depth[i])
            mask += [w - (1 << 64) if w >> 63 else w for w in words] if parents else []
            cu.append(cu[b] + m)
            self.lens[b] += m
        return cu, seq, pos, slots, mask

    def truncate(self, lengths):
        gone = []
        for b, (L, k) in enumerate(zip(self.lens, lengths)):
            for p in range(-(-min(L, k) // PAGE), -(-L // PAGE)):
                gone.append(self.table[b][p])
                if self.free is not None:
                    self.table[b][p] = -1
            self.lens[b] = min(L, k)
        if self.free is not None:
            self.free += gone[::-1]


def state_of(cache):
    free = None if cache.free is None else cache.free.tolist()
    return cache.page_table.tolist(), cache.seqlens.tolist(), None if free is None else free[1:1 + free[0]]


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def random_parents(r, new):
    return [r.randint(max(-1, i - 5), i - 1) for m in new for i in range(m)]


# ------------------------------------------------------------------------------------------------ refusals (no GPU)
@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def test_c_entries_refuse_bad_arguments(lib):
    pg = lambda **k: ctypes.byref(_lib.Pages(*[k.get(n, d) for n, d in (("t", 4096), ("l", 8192), ("f", 0), ("b", 2), ("m", 4), ("n", 8))]))
    plan = lambda **k: ctypes.byref(_lib.Plan(*[k.get(n, 4096) for n in ("cu", "seq", "pos", "slots", "mask", "ticket")], 0, k.get("cap", 4)))
    assert lib.pkv_plan_step(None, 1024, None, plan(), None) == -1
    assert lib.pkv_plan_step(pg(t=0), 1024, None, plan(), None) == -1
    assert lib.pkv_plan_step(pg(m=0), 1024, None, plan(), None) == -1
    assert lib.pkv_plan_step(pg(b=-1), 1024, None, plan(), None) == -1
    assert lib.pkv_plan_step(pg(b=4097), 1024, None, plan(), None) == -2
    assert lib.pkv_plan_step(pg(n=1 << 25), 1024, None, plan(), None) == -2            # slots past 31 bits
    assert lib.pkv_plan_step(pg(), None, None, plan(), None) == -1
    assert lib.pkv_plan_step(pg(), 1024, None, None, None) == -1
    assert lib.pkv_plan_step(pg(), 1024, None, plan(ticket=0), None) == -1
    assert lib.pkv_plan_step(pg(), 1024, 1024, plan(mask=0), None) == -1               # parents without room for masks
    assert lib.pkv_plan_step(pg(), 1024, None, plan(cap=-1), None) == -1
    assert lib.pkv_plan_step(pg(), 1024, None, plan(cap=1 << 30), None) == -2
    assert lib.pkv_truncate(pg(), None, None, None) == -1
    assert lib.pkv_truncate(pg(), 8192, None, None) == -1                              # the lengths themselves
    cache = _lib.Cache(4096, 4096, 8, 256, 8, 128)
    layers = lambda *c: (ctypes.c_void_p * len(c))(*[ctypes.addressof(x) for x in c])
    keep = lambda arr, n, p=None, cap=4, out=None: lib.pkv_keep_rows(arr, n, p or pg(), 1024, cap, 1024, 1024, out, None, None)
    assert keep(None, 1) == -1 and keep(layers(cache), 0) == -1 and keep(layers(cache), 1, cap=-1) == -1
    assert keep(layers(cache), 1, out=8192) == -1
    assert keep(layers(cache, cache), 2) == -1                                          # a pool twice
    assert keep(layers(_lib.Cache(4096, 4096, 8, 250, 8, 128)), 1) == -2
    assert keep(layers(_lib.Cache(4096, 4096, 7, 256, 8, 128)), 1) == -1                # a pool smaller than the table's
    assert keep(layers(_lib.Cache(4096, 4100, 8, 256, 8, 128)), 1) == -1                # misaligned values


def test_python_calls_refuse_bad_tensors(lib):
    cache = PagedLatentCache(256, 8, 128, 2, 512, "cpu")
    plan = cache.step_plan(6)
    n = torch.ones(2, dtype=torch.int32)
    for bad in (n.long(), n[:1], torch.ones((2, 1), dtype=torch.int32), torch.ones(4, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError):
            cache.plan_step(plan, bad)
        with pytest.raises(ValueError):
            cache.truncate(bad)
        with pytest.raises(ValueError):
            cache.keep_rows(plan, torch.zeros(6, dtype=torch.int32), bad)
    with pytest.raises(ValueError):
        cache.plan_step(plan, n, parents=torch.zeros(6, dtype=torch.int32))             # a plan without masks
    with pytest.raises(ValueError):
        cache.plan_step(cache.step_plan(6, tree=True), n, parents=torch.zeros(5, dtype=torch.int32))
    with pytest.raises(ValueError):
        cache.keep_rows(plan, torch.zeros(5, dtype=torch.int32), n)
    with pytest.raises(ValueError):
        cache.step_plan(-1)
    other = PagedLatentCache(256, 8, 128, 3, 512, "cpu")
    with pytest.raises(ValueError):
        other.plan_step(plan, torch.ones(3, dtype=torch.int32))                         # a plan of another batch
    with pytest.raises(ValueError):
        other.share_pages(cache)
    with pytest.raises(ValueError):
        cache.keep_rows(plan, torch.zeros(6, dtype=torch.int32), n, layers=[PagedLatentCache(256, 8, 128, 2, 512, "cpu")])


def test_page_pool_and_sharing_on_the_host(lib):
    a, b = (PagedLatentCache(256, 8, 128, 2, 512, "cpu") for _ in range(2))
    a.use_page_pool()
    assert a.free.tolist() == [8, 7, 6, 5, 4, 3, 2, 1, 0] and int(a.page_table.max()) == -1
    b.share_pages(a)
    assert b.page_table is a.page_table and b.seqlens is a.seqlens and b.free is a.free


# ------------------------------------------------------------------------------------------------ on the GPU
def check_plan(cache, ref, plan, new, cap, parents=None):
    before = [t.clone() for t in (plan.seq, plan.positions)] + [None if plan.mask is None else plan.mask.clone()]
    cache.plan_step(plan, i32(new), parents=None if parents is None else i32(parents + [7] * (cap - len(parents))))
    want = ref.plan(new, cap, parents)
    cu, seq, pos, slots, mask = want if want else ([0] * (len(new) + 1), [], [], [], [])
    n = len(seq)
    assert plan.cu.tolist() == cu
    assert plan.seq[:n].tolist() == seq and plan.positions[:n].tolist() == pos
    assert plan.slots.tolist() == slots + [-1] * (cap - n)
    if parents is not None:
        assert plan.mask[:n].tolist() == mask
    for t, old in zip((plan.seq, plan.positions, plan.mask), before):
        if t is not None:
            assert torch.equal(t[n:], old[n:])                                          # behind the last token: as they were
    assert state_of(cache) == (ref.table, ref.lens, ref.free)
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("batch,max_tokens,top,tree", [
    (1, 128, 1, False), (1, 1024, 64, True), (3, 700, 300, False), (7, 1100, 64, True), (64, 2000, 1, False),
    (130, 900, 33, True), (5, 40000, 12000, False), (1500, 256, 5, True), (4096, 256, 3, False)])
def test_plan_and_truncate_against_lists(batch, max_tokens, top, tree):
    r = random.Random(batch * 7 + top)
    cache = PagedLatentCache(128, 1, 128, batch, max_tokens, "cuda", with_v=False, n_pages=batch * (-(-max_tokens // PAGE)) + 1)
    cache.use_page_pool()
    order = list(range(cache.n_pages))
    r.shuffle(order)
    cache.free[1:] = i32(order)
    ref = Tables(*state_of(cache))
    cap = batch * top + 5
    plan = cache.step_plan(cap, tree=tree)
    for step in range(6):
        new = [r.choice([0, 1, top, r.randint(0, top)]) for _ in range(batch)]
        new = [min(m, cache.max_pages * PAGE - L) for m, L in zip(new, ref.lens)]
        assert check_plan(cache, ref, plan, new, cap, random_parents(r, new) if tree else None)
        lengths = [r.choice([L, max(0, L - 1), L + 9, r.randint(0, L)]) for L in ref.lens] if step != 3 else [0] * batch
        cache.truncate(i32(lengths))
        ref.truncate(lengths)
        assert state_of(cache) == (ref.table, ref.lens, ref.free)
    assert int(plan.status.abs().sum()) == 0 and int(cache.status.abs().sum()) == 0 and int(plan.ticket) == 0


@pytest.mark.gpu
def test_plan_on_the_fixed_mapping():
    cache = PagedLatentCache(128, 1, 128, 3, 512, "cuda", with_v=False)
    ref = Tables(*state_of(cache))
    plan = cache.step_plan(600)
    for new in ([130, 0, 256], [1, 1, 1], [3, 500, 0]):
        assert check_plan(cache, ref, plan, new, 600)
    cache.truncate(i32([128, 0, 257]))
    ref.truncate([128, 0, 257])
    assert state_of(cache) == (ref.table, ref.lens, None)


@pytest.mark.gpu
@pytest.mark.parametrize("big", [False, True])                                          # one CTA, and several
def test_refused_steps_change_nothing(big):
    cap = 5000 if big else 40
    cache = PagedLatentCache(128, 1, 128, 4, 512, "cuda", with_v=False, n_pages=6)
    cache.use_page_pool()
    ref = Tables(*state_of(cache))
    plan = cache.step_plan(cap, tree=True)
    assert check_plan(cache, ref, plan, [3, 0, 30, 1], cap, [-1, 0, 0] + [i - 1 for i in range(30)] + [-1])
    for new, parents, code in [([-1, 1, 1, 1], None, 4), ([1, 1, 510, 1], None, 4), ([0, 400, 0, 0], None, 5),
                               ([40, 1, 0, 0], None, 4 if not big else 0), ([65, 0, 0, 0], [-1] * 65, 4),
                               ([2, 2, 0, 0], [-1, 0, -1, 1], 4), ([2, 0, 0, 2], [-1, 0, -2, 0], 4), ([1 << 30, 1 << 30, 1 << 30, 1 << 30], None, 4)]:
        plan.status.zero_()
        if code:
            plan.seq.fill_(3)
            before = state_of(cache)
            p = None if parents is None else i32((parents + [0] * cap)[:cap])
            cache.plan_step(plan, i32(new), parents=p)
            assert plan.cu.tolist() == [0] * 5 and set(plan.slots.tolist()) == {-1}
            assert state_of(cache) == before and set(plan.seq.tolist()) == {3}
            assert int(plan.status[0]) == code, (new, plan.status.tolist())
        else:
            assert check_plan(cache, ref, plan, new, cap)
    before = state_of(cache)
    cache.truncate(i32([0, -1, 0, 0]))
    assert state_of(cache) == before and int(cache.status[0]) == 4
    assert int(plan.ticket) == 0


@pytest.mark.gpu
def test_plan_without_room_or_tokens():
    cache = PagedLatentCache(128, 1, 128, 2, 512, "cuda", with_v=False)
    plan = cache.step_plan(0)
    cache.plan_step(plan, i32([0, 0]))
    assert plan.cu.tolist() == [0, 0, 0] and int(plan.status[0]) == 0
    cache.plan_step(plan, i32([1, 0]))
    assert int(plan.status[0]) == 4 and cache.seqlens.tolist() == [0, 0]


@pytest.mark.gpu
def test_planned_step_in_a_captured_graph():
    """Lengths live on the device: one captured plan + truncate serves every replay, on a stream of its own."""
    cache = PagedLatentCache(128, 1, 128, 9, 4000, "cuda", with_v=False)
    cache.use_page_pool()
    ref = Tables(*state_of(cache))
    plan, n_new, lengths = cache.step_plan(9 * 600), i32([0] * 9), i32([0] * 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        cache.plan_step(plan, n_new)
        cache.truncate(lengths)
    r = random.Random(4)
    for _ in range(8):
        new = [r.randint(0, 600) for _ in range(9)]
        cut = [r.randint(0, L + m) for L, m in zip(ref.lens, new)]
        n_new.copy_(i32(new)), lengths.copy_(i32(cut))
        g.replay()
        want = ref.plan(new, 5400)
        ref.truncate(cut)
        assert plan.slots[:len(want[3])].tolist() == want[3] and state_of(cache) == (ref.table, ref.lens, ref.free)


def fill(cache, r):
    gen = torch.Generator(device="cuda").manual_seed(r.randrange(1 << 30))
    pools = [cache.latent] + [p.view(-1).view(torch.uint8) for p in (cache.v, cache.vq) if p is not None]
    for p in pools:
        p.copy_(torch.randint(0, 256, p.shape, generator=gen, device="cuda", dtype=torch.uint8))
    return pools


def rows_of(cache, slots):
    """Every byte of the rows at `slots`, through the cache's own readers: (codes, scales, values ...)."""
    if not slots.numel():
        return ()
    _, codes, scales = cache.read(slots, 1.0, rows=False)
    if cache.v_bits:
        _, c, s = cache.read_vq(slots)
        return codes, scales, c, s.view(torch.int16)
    return (codes, scales) if cache.v is None else (codes, scales, cache.v_rows(slots).view(torch.int16))


@pytest.mark.gpu
@pytest.mark.parametrize("shapes,base,n,v_bits", [
    ([(256, 8, 128)], [0], [1], 0), ([(256, 8, 128)], [120, 0, 500], [64, 64, 33], 0), ([(128, 32, 128)], [127, 63], [5, 64], 0),
    ([(256, 8, 128), (240, 8, 128), (112, 4, 128)], [200, 3], [20, 64], 3), ([(144, 2, 64)], [90], [50], 0),
    ([(256, 1, 128)] * 50, [126, 10, 255], [9, 2, 64], 2), ([(64, 3, 8)], [100, 1], [40, 0], 0)])
def test_kept_rows_move_byte_for_byte(shapes, base, n, v_bits):
    r = random.Random(sum(base) + len(shapes))
    B, most = len(base), max(b + m for b, m in zip(base, n)) + 1
    caches = [PagedLatentCache(W, g, d, B, most, "cuda", v_bits=v_bits, with_v=True) for W, g, d in shapes]
    caches[0].use_page_pool()
    for c in caches[1:]:
        c.share_pages(caches[0])
    lead = caches[0]
    plan = lead.step_plan(sum(n) + 3)
    lead.plan_step(lead.step_plan(sum(base)), i32(base))
    lead.plan_step(plan, i32(n))
    for round_ in range(3):
        pools = [fill(c, r) for c in caches]
        kept = [sorted(r.sample(range(m), r.choice([0, m, r.randint(0, m)]) if round_ else m // 2)) for m in n]
        keep = [-5] * (sum(n) + 3)
        for b, k in enumerate(kept):
            keep[int(plan.cu[b]):int(plan.cu[b]) + len(k)] = k
        slots = [plan.slots[int(plan.cu[b]):int(plan.cu[b + 1])] for b in range(B)]
        src = torch.cat([s[i32(k).long()] for s, k in zip(slots, kept)])
        dst = torch.cat([s[:len(k)] for s, k in zip(slots, kept)])
        want = [[t.clone() for t in rows_of(c, src)] for c in caches]
        stay = torch.tensor(sorted(set(range(lead.n_pages * PAGE)) - set(dst.tolist())), dtype=torch.int32, device="cuda")
        others = [[t.clone() for t in rows_of(c, stay)] for c in caches]
        lengths = torch.full((B,), -7, dtype=torch.int32, device="cuda")
        lead.keep_rows(plan, i32(keep), i32([len(k) for k in kept]), lengths, layers=caches)
        assert lengths.tolist() == [b + len(k) for b, k in zip(base, kept)]
        assert lead.seqlens.tolist() == [b + m for b, m in zip(base, n)]
        for c, w, o in zip(caches, want, others):
            assert all(torch.equal(x, y) for x, y in zip(rows_of(c, dst), w))
            assert all(torch.equal(x, y) for x, y in zip(rows_of(c, stay), o))           # nothing else is touched
        del pools
    assert int(lead.status.abs().sum()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("keep,n_keep", [([2, 1, 0], 2), ([1, 1, 0], 2), ([0, 3, 0], 2), ([-1, 0, 0], 1), ([0, 1, 2], 4), ([0, 1, 2], -1)])
def test_refused_paths_leave_their_sequence_alone(keep, n_keep):
    cache = PagedLatentCache(256, 2, 128, 2, 400, "cuda")
    cache.seqlens.copy_(i32([130, 10]))
    plan = cache.step_plan(6)
    cache.plan_step(plan, i32([3, 3]))
    pools = fill(cache, random.Random(1))
    before = [p.clone() for p in pools]
    lengths = i32([0, 0])
    cache.keep_rows(plan, i32(keep + [1, 2, 0]), i32([n_keep, 2]), lengths)
    assert lengths.tolist() == [133, 12] and cache.status[:2].tolist() == [4, 0]
    cache.status.zero_()
    moved = plan.slots[3:5].long()
    other = PagedLatentCache(256, 2, 128, 2, 400, "cuda")
    other.latent.copy_(before[0]), other.v.view(-1).view(torch.uint8).copy_(before[1])
    rest = torch.tensor(sorted(set(range(cache.n_pages * PAGE)) - set(moved.tolist())), dtype=torch.int32, device="cuda")
    assert all(torch.equal(x, y) for x, y in zip(rows_of(cache, rest), rows_of(other, rest)))


def test_c_entries_refuse_an_array_given_twice(lib):
    """Other CTAs still read the inputs when the first writes its results."""
    pg, cache = _lib.Pages(4096, 8192, 0, 2, 4, 8), _lib.Cache(4096, 4096, 8, 256, 8, 128)
    for twice in (1024, 2048, 5120, 6144):
        plan = _lib.Plan(1024, 2048, 5120, 6144, 7168, 9216, 0, 4)
        assert lib.pkv_plan_step(ctypes.byref(pg), twice, None, ctypes.byref(plan), None) == -1
        assert lib.pkv_plan_step(ctypes.byref(pg), 10240, twice, ctypes.byref(plan), None) == -1
    one = (ctypes.c_void_p * 1)(ctypes.addressof(cache))
    for out in (1024, 2048, 5120, 8192):
        assert lib.pkv_keep_rows(one, 1, ctypes.byref(pg), 1024, 4, 2048, 5120, out, None, None) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[5, 0, 64], [1, 1, 1], [700, 63, 900]])
def test_a_plan_with_masks_has_a_chains_without_parents(new):
    """Nothing of an earlier tree stays in the words: each token sees itself and the step's tokens before it."""
    cache = PagedLatentCache(128, 1, 128, 3, 2000, "cuda", with_v=False)
    cap = sum(new) + 4
    plan = cache.step_plan(cap, tree=True)
    plan.mask.fill_(0x5a5a)
    cache.plan_step(plan, i32(new))
    words = [(1 << min(i + 1, 64)) - 1 for m in new for i in range(m)]
    assert plan.mask.tolist() == [w - (1 << 64) if w >> 63 else w for w in words] + [0x5a5a] * 4
    assert plan.positions[:sum(new)].tolist() == [i for m in new for i in range(m)] and int(plan.status[0]) == 0


@pytest.mark.parametrize("out", ["cu", "seq", "positions", "slots", "mask", "ticket", "status"])
@pytest.mark.parametrize("shift", [-4, 0, 4])
def test_c_entries_refuse_arrays_that_overlap(lib, out, shift):
    """An input that begins inside a result, or reaches into it, is written while other CTAs still read it."""
    pg = _lib.Pages(4096, 8192, 0, 2, 4, 8)
    at = dict(cu=(0x10000, 12), seq=(0x20000, 32), positions=(0x30000, 32), slots=(0x40000, 32), mask=(0x50000, 64), ticket=(0x60000, 4), status=(0x70000, 16))
    plan = _lib.Plan(*[at[k][0] for k in ("cu", "seq", "positions", "slots", "mask", "ticket", "status")], 8)
    begin, size = at[out]
    inside = begin + size - 4 if shift > 0 else begin + shift                     # its last word; itself; an array that ends in its first word
    assert lib.pkv_plan_step(ctypes.byref(pg), inside, None, ctypes.byref(plan), None) == -1
    assert lib.pkv_plan_step(ctypes.byref(pg), 0x9000, inside, ctypes.byref(plan), None) == -1


@pytest.mark.parametrize("shift", [-4, 0, 4])
def test_c_entries_refuse_lengths_that_overlap(lib, shift):
    pg, cache = _lib.Pages(0x10000, 0x20000, 0x30000, 2, 4, 8), _lib.Cache(4096, 4096, 8, 256, 8, 128)
    one = (ctypes.c_void_p * 1)(ctypes.addressof(cache))
    for begin, size in ((0x10000, 32), (0x20000, 8), (0x30000, 36)):              # table, lengths, pool
        inside = begin + size - 4 if shift > 0 else begin + shift
        assert lib.pkv_truncate(ctypes.byref(pg), inside, None, None) == -1
    for begin, size in ((0x10000, 32), (0x20000, 8), (0x40000, 12), (0x50000, 16), (0x60000, 8)):          # .. cu, keep, n_keep
        inside = begin + size - 4 if shift > 0 else begin + shift
        assert lib.pkv_keep_rows(one, 1, ctypes.byref(pg), 0x40000, 4, 0x50000, 0x60000, inside, None, None) == -1


@pytest.mark.gpu
def test_the_first_problem_stays_until_it_is_cleared():
    """Both status words tell of one problem, however many there are."""
    cache = PagedLatentCache(128, 1, 128, 3, 512, "cuda", with_v=False, n_pages=4)
    cache.use_page_pool()
    plan = cache.step_plan(2000)
    cache.plan_step(plan, i32([1, -1, 1]))
    assert plan.status[:2].tolist() == [4, 1]
    cache.plan_step(plan, i32([512, 512, 512]))                                   # eight pages missing
    assert plan.status[:2].tolist() == [4, 1]
    plan.status.zero_()
    cache.plan_step(plan, i32([512, 512, 512]))
    assert plan.status[:2].tolist() == [5, 8]
    cache.truncate(i32([0, 0, -1]))
    cache.truncate(i32([-1, 0, 0]))
    assert cache.status[:2].tolist() == [4, 2]
