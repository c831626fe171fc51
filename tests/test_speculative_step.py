"""The operators of a speculative step together, as a patched layer runs them: drafts planned, written, attended to, a path kept,
and decoding going on from there -- against the same tokens decoded one by one.

Tolerance: the token-by-token outputs are within 2e-3 of the formula in the 2-norm (what decode attention is held to), the
drafted ones within 5e-3 (two roundings to bf16 of at most 2^-8, uniform: 3.2e-3, and the logits' share). The two write paths form
a row's sums in another order, so a latent may differ in its last bit and, at a tie, in one code: far below 1e-3. In all 8e-3."""
import random
import types

import pytest
import torch

from phasorkv_b200 import PhasorKey, PhasorKeyPatch, synth
from phasorkv_b200.patch import LayerDecodeState

from test_tree_attn import Case

pytestmark = pytest.mark.gpu
NORM = 8e-3
D = 256


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def state(pk, B, v_bits, x, v):
    st = LayerDecodeState(pk, B, 512, v_bits=v_bits)
    st.calibrated = pk.second_blocks is not None
    st.prefill(x, v)
    return st


@pytest.mark.parametrize("config,v_bits,other", [("cfg2", 0, None), ("cfg3", 0, None), ("cfg5", 0, None), ("cfg2", 3, None),
                                                 ("cfg2", 0, "attn_scale"), ("cfg2", 0, "tiers"), ("cfg3", 2, "tiers")])
@pytest.mark.parametrize("kind", ["tree", "chain"])
def test_verified_drafts_match_tokens_decoded_one_by_one(config, v_bits, other, kind):
    spec = synth.make_layer(config, 0, d_model=D, factor_gain=16.0)
    if other == "attn_scale":
        spec.attn_scale = 1.3
    pk = PhasorKey.from_spec(spec)
    B, T, n = 3, 122, 11                                             # the drafts cross a page
    g, r = torch.Generator(device="cuda").manual_seed(5), random.Random(5)
    t = lambda *s: torch.randn(s, generator=g, device="cuda")
    x0, v0 = t(B, T, D), t(B, T, spec.n_kv, 128).to(torch.bfloat16)
    if other == "tiers":                                             # one scale per 16-aligned span instead of the calibrated one
        W = pk.cache_width
        edges = [0, 32, 112, W]
        pk.set_second_tiers([(a, b, 0.01 * 3 ** i) for i, (a, b) in enumerate(zip(edges, edges[1:]))])
    one, many = state(pk, B, v_bits, x0, v0), state(pk, B, v_bits, x0, v0)
    for round_ in range(3):
        x, q, v = t(B, n, D), t(B, n, spec.n_q, 128), t(B, n, spec.n_kv, 128).to(torch.bfloat16)
        parents = [[i - 1 if kind == "chain" else r.randint(max(-1, i - 4), i - 1) for i in range(n)] for _ in range(B)]
        out = many.verify(x, q, v, None if kind == "chain" else torch.tensor(parents))
        with pytest.raises(RuntimeError):
            many.decode(x[:, 0], q[:, 0], v[:, 0])
        # a path of the same length in every sequence (the plain decode steps all sequences together)
        paths = []
        for b in range(B):
            path = [r.randrange(n)]
            while parents[b][path[0]] >= 0:
                path.insert(0, parents[b][path[0]])
            paths.append(path)
        k = min(map(len, paths)) if round_ != 1 else 0
        paths = [p[:k] for p in paths]
        many.accept(paths)
        for j in range(k):
            pick = lambda a: torch.stack([a[b, paths[b][j]] for b in range(B)])
            want = one.decode(pick(x), pick(q), pick(v))
            assert rel(pick(out), want) < NORM, (round_, j)
        assert one.lengths == many.lengths and many.cache.seqlens.tolist() == many.lengths
        x, q, v = t(B, D), t(B, spec.n_q, 128), t(B, spec.n_kv, 128).to(torch.bfloat16)
        assert rel(many.decode(x, q, v), one.decode(x, q, v)) < NORM
    for s in (many.ws, many.cache, *[w[1] for w in many.tree.values()], *[w[0] for w in many.tree.values()]):
        assert int(s.status.abs().sum()) == 0


def test_patched_layer_verifies_and_accepts():
    """Through the patched forward of an attention module: drafts in one pass, then the path in every layer."""
    spec = synth.make_layer("cfg2", 0, d_model=D, factor_gain=16.0)
    g = torch.Generator(device="cuda").manual_seed(2)
    lin = lambda i, o: torch.nn.Linear(i, o, bias=False, device="cuda", dtype=torch.float32)

    class Attn(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.head_dim = 128
            self.q_proj, self.v_proj, self.o_proj = lin(D, 32 * 128), lin(D, 8 * 128), lin(32 * 128, D)

        def forward(self, hidden_states, **kw):
            return hidden_states, None
    layers = [types.SimpleNamespace(self_attn=Attn()) for _ in range(2)]
    patch = PhasorKeyPatch(install_forward=True, max_tokens=512)
    undo = [patch.patch(i, y, spec, 8, 128, 32, "cuda") for i, y in enumerate(layers)]
    h = lambda n: torch.randn((2, n, D), generator=g, device="cuda")
    prompt, drafts = h(40), h(4)
    with torch.no_grad():
        for y in layers:
            y.self_attn(prompt)
            y.self_attn.kv_tree = torch.tensor([[-1, 0, 0, 2], [-1, -1, 1, 2]])
        tree = [y.self_attn(drafts)[0] for y in layers]
        for y in layers:
            y.self_attn.kv_tree = None
        patch.accept([[0, 2, 3], [1, 2, 3]])
        assert all(st.lengths == [43, 43] for st in patch.states.values())
        after = [y.self_attn(h(1))[0] for y in layers]
        patch.reset()
        for i, y in enumerate(layers):
            y.self_attn(prompt)
            for j in range(3):
                step = torch.stack([drafts[0, [0, 2, 3][j]], drafts[1, [1, 2, 3][j]]])[:, None]
                got = torch.stack([tree[i][0, [0, 2, 3][j]], tree[i][1, [1, 2, 3][j]]])
                assert rel(got, y.self_attn(step)[0][:, 0]) < NORM
    assert all(a.isfinite().all() for a in after)
    for u in undo:
        u()


def test_refusals_of_a_layer_state():
    pk = PhasorKey.from_spec(synth.make_layer("cfg2", 0, d_model=D))
    t = lambda *s: torch.randn(s, device="cuda")
    st = state(pk, 2, 0, t(2, 500, D), t(2, 500, 8, 128).to(torch.bfloat16))
    with pytest.raises(RuntimeError):
        st.accept([[], []])
    for B, n, parents in ((3, 4, None), (2, 65, None), (2, 0, None), (2, 2, [[-1, 1], [-1, 0]]), (2, 2, [[-2, 0], [-1, 0]]), (2, 2, [[-1], [0]])):
        with pytest.raises(ValueError):
            st.verify(t(B, n, D), t(B, n, 32, 128), t(B, n, 8, 128), None if parents is None else torch.tensor(parents))
    with pytest.raises(RuntimeError):
        st.verify(t(2, 13, D), t(2, 13, 32, 128), t(2, 13, 8, 128))      # 512 tokens per sequence
    st.verify(t(2, 4, D), t(2, 4, 32, 128), t(2, 4, 8, 128))
    with pytest.raises(RuntimeError):
        st.verify(t(2, 4, D), t(2, 4, 32, 128), t(2, 4, 8, 128))
    for bad in ([[0]], [[0], [4]], [[1, 0], []], [[0, 0], []], [[-1], []], [[1, 2], []], [[0, 2], []]):
        with pytest.raises(ValueError):
            st.accept(bad)
    st.accept([[0, 1], []])
    assert st.lengths == [502, 500] and st.cache.seqlens.tolist() == [502, 500]


@pytest.mark.parametrize("fails", ["write_paged", "tree_step"])
def test_a_verification_that_fails_leaves_the_layer_as_it_was(fails, monkeypatch):
    """An error behind the plan: the drafts are no cached tokens, and the next verification gives what it would have given."""
    pk = PhasorKey.from_spec(synth.make_layer("cfg2", 0, d_model=D, factor_gain=16.0))
    g = torch.Generator(device="cuda").manual_seed(3)
    t = lambda *s: torch.randn(s, generator=g, device="cuda")
    x0, v0 = t(2, 126, D), t(2, 126, 8, 128)
    x, q, v = t(2, 5, D), t(2, 5, 32, 128), t(2, 5, 8, 128)
    st, other = state(pk, 2, 0, x0, v0), state(pk, 2, 0, x0, v0)

    def error(*a, **k):
        raise RuntimeError("out of memory")
    with monkeypatch.context() as m:
        m.setattr(pk, fails, error)
        with pytest.raises(RuntimeError, match="out of memory"):
            st.verify(x, q, v)
    assert st.cache.seqlens.tolist() == st.lengths == [126, 126] and st.drafted is None
    assert torch.equal(st.verify(x, q, v), other.verify(x, q, v))
    st.accept([[0], []])
    assert st.cache.seqlens.tolist() == st.lengths == [127, 126]


def patched_layers(k):
    """k attention layers with patched forwards -> (layers, their undo calls, the patch)"""
    spec = synth.make_layer("cfg2", 0, d_model=D, factor_gain=16.0)
    lin = lambda i, o: torch.nn.Linear(i, o, bias=False, device="cuda", dtype=torch.float32)

    class Attn(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.head_dim = 128
            self.q_proj, self.v_proj, self.o_proj = lin(D, 32 * 128), lin(D, 8 * 128), lin(32 * 128, D)

        def forward(self, hidden_states, **kw):
            return hidden_states, None
    layers = [types.SimpleNamespace(self_attn=Attn()) for _ in range(k)]
    patch = PhasorKeyPatch(install_forward=True, max_tokens=512)
    return layers, [patch.patch(i, y, spec, 8, 128, 32, "cuda") for i, y in enumerate(layers)], patch


def test_layers_and_draft_counts_share_their_scratch():
    """The workspaces of verification are the larger part of its memory: one buffer for all layers of a patch, whatever their draft counts."""
    layers, undo, patch = patched_layers(3)
    g = torch.Generator(device="cuda").manual_seed(7)
    h = lambda n: torch.randn((2, n, D), generator=g, device="cuda")
    with torch.no_grad():
        for y in layers:
            y.self_attn(h(20))
            y.self_attn.kv_tree = "chain"
        before = torch.cuda.memory_allocated()
        for n in (1, 2, 3, 5, 8, 13, 21, 34, 64, 7):
            drafts = h(n)
            for y in layers:
                y.self_attn(drafts)
            patch.accept([[], [0]])
    spaces = [w[1] for st in patch.states.values() for w in st.tree.values()]
    assert len(spaces) == 30 and len({w.buffer.data_ptr() for w in spaces}) == 1
    largest = max(w.bytes for w in spaces)
    assert torch.cuda.memory_allocated() - before < 1.5 * largest          # the rest: plans and results, a few hundred KB
    for u in undo:
        u()


def test_a_shared_workspace_that_grew_still_serves_the_small_steps():
    """Draft counts up and down over layers that share their scratch: the outputs are those of layers of their own."""
    pk = PhasorKey.from_spec(synth.make_layer("cfg2", 0, d_model=D, factor_gain=16.0))
    g = torch.Generator(device="cuda").manual_seed(8)
    t = lambda *s: torch.randn(s, generator=g, device="cuda")
    x0, v0 = t(2, 100, D), t(2, 100, 8, 128)
    shared, own = [state(pk, 2, 0, x0, v0) for _ in range(2)], [state(pk, 2, 0, x0, v0) for _ in range(2)]
    shared[1].scratch = shared[0].scratch
    for n in (2, 40, 2, 64, 1, 40):
        x, q, v = t(2, n, D), t(2, n, 32, 128), t(2, n, 8, 128)
        for a, b in zip(shared, own):
            assert torch.equal(a.verify(x, q, v), b.verify(x, q, v))
            a.accept([[0], []]), b.accept([[0], []])


def test_paths_of_different_lengths():
    """Sequences that accept different numbers of rows, none among them: what follows is what each alone would have given."""
    pk = PhasorKey.from_spec(synth.make_layer("cfg2", 0, d_model=D, factor_gain=16.0))
    B, T, n = 3, 121, 7
    g, r = torch.Generator(device="cuda").manual_seed(6), random.Random(6)
    t = lambda *s: torch.randn(s, generator=g, device="cuda")
    x0, v0 = t(B, T, D), t(B, T, 8, 128).to(torch.bfloat16)
    many, alone = state(pk, B, 0, x0, v0), []
    for b in range(B):
        st = LayerDecodeState(pk, 1, 512)
        st.calibrated = True                                         # one scale for all: the batch's
        st.prefill(x0[b:b + 1], v0[b:b + 1])
        alone.append(st)
    for round_ in range(4):
        x, q, v = t(B, n, D), 20 * t(B, n, 32, 128), t(B, n, 8, 128).to(torch.bfloat16)      # logits of a few units
        parents = [[r.randint(max(-1, i - 3), i - 1) for i in range(n)] for _ in range(B)]
        out = many.verify(x, q, v, torch.tensor(parents))
        paths = []
        for b in range(B):
            path = [r.randrange(n)]
            while parents[b][path[0]] >= 0:
                path.insert(0, parents[b][path[0]])
            paths.append(path[:[0, 1, n][(b + round_) % 3]])
        many.accept(paths)
        for b, path in enumerate(paths):
            for j in path:
                want = alone[b].decode(x[b:b + 1, j], q[b:b + 1, j], v[b:b + 1, j])
                assert rel(out[b, j], want[0]) < NORM, (round_, b, j)
        assert many.lengths == [st.lengths[0] for st in alone] and many.cache.seqlens.tolist() == many.lengths
    assert len(set(many.lengths)) == 3


def test_ragged_trees_over_layers_that_share_a_page_pool():
    """The operators together, as a server runs them: one plan a step for all layers, drafts written and attended to in each, one move of
    the accepted rows, the pages behind them back. Outputs against the formula in 64 bits, the caches byte for byte against
    what was accepted so far, and no page lost."""
    specs = [(synth.make_layer("cfg2", 0, d_model=D, factor_gain=16.0), 0), (synth.make_layer("cfg3", 1, d_model=D, factor_gain=16.0), 3),
             (synth.make_layer("cfg2", 2, d_model=D, factor_gain=16.0), 2)]
    pks = [PhasorKey.from_spec(s) for s, _ in specs]
    B, most, r = 5, 700, random.Random(12)
    g = torch.Generator(device="cuda").manual_seed(12)
    t = lambda *s: torch.randn(s, generator=g, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    caches = [pk.new_cache(B, most, v_bits=bits) for pk, (_, bits) in zip(pks, specs)]
    lead = caches[0]
    for c in caches[1:]:
        c.share_pages(lead)
    lead.use_page_pool()
    for pk in pks:
        pk.set_second(0.002)
    cap = B * 20 + 7
    plan, prompts, n_keep, lengths = lead.step_plan(cap, tree=True), lead.step_plan(B * 300), i32([0] * B), i32([0] * B)
    spaces = [pk.tree_workspace(B, cap, 20, most) for pk in pks]
    out = torch.zeros((cap, 32, 128), dtype=torch.bfloat16, device="cuda")

    def write(p, n):                                                 # random inputs of n planned tokens, and of the rows behind them
        for pk, c in zip(pks, caches):
            pk.write_paged(c, t(p.capacity, D), p.positions, p.slots, v=t(p.capacity, 8, 128).to(torch.bfloat16))

    def rows(c, slots):
        codes, scales = c.read(slots, 0.002, rows=False)[1:]
        return [codes, scales] + ([x.view(torch.int16) if x.dtype is torch.bfloat16 else x for x in c.read_vq(slots)[1:]] if c.v_bits else [c.v_rows(slots).view(torch.int16)])

    def place(b, lo, hi):
        return lead.slots(i32([b] * (hi - lo)), i32(list(range(lo, hi))))

    base = [300, 0, 127, 128, 61]
    lead.plan_step(prompts, i32(base))
    write(prompts, sum(base))
    kept = [[rows(c, place(b, 0, base[b])) for b in range(B)] for c in caches]
    for round_ in range(6):
        n = [r.choice([0, 1, 20, r.randint(0, 20)]) for _ in range(B)]
        chain = round_ == 4                                          # planned without parents where trees were before
        parents = [[i - 1 if chain else r.randint(max(-1, i - 4), i - 1) for i in range(m)] for m in n]
        flat = sum(parents, [])
        lead.plan_step(plan, i32(n), parents=None if chain else i32(flat + [-1] * (cap - len(flat))))
        write(plan, sum(n))
        words, positions = [], []
        for b, m in enumerate(n):
            w, d = [], []
            for i, p in enumerate(parents[b]):
                w.append((w[p] if p >= 0 else 0) | 1 << i)
                d.append(d[p] + 1 if p >= 0 else 0)
            words.append(w), positions.append([base[b] + k for k in d])
        for pk, c, ws in zip(pks, caches, spaces):
            q = 20 * t(cap, 32, 128)                                 # logits of a few units
            out.fill_(7.0)
            pk.tree_step(c, q, plan, ws, out=out)
            case = object.__new__(Case)
            case.pk, case.cache, case.q, case.ws, case.base, case.n, case.words, case.positions = pk, c, q, ws, base, n, words, positions
            case.check(out)
            assert (out[sum(n):] == 7).all()
        paths = []
        for b, m in enumerate(n):
            path = [r.randrange(m)] if m and r.random() < 0.8 else []
            while path and parents[b][path[0]] >= 0:
                path.insert(0, parents[b][path[0]])
            paths.append(path)
        cu = plan.cu.tolist()
        for l, c in enumerate(caches):
            for b, path in enumerate(paths):
                if path:
                    new = rows(c, plan.slots[i32([cu[b] + i for i in path]).long()])
                    kept[l][b] = [torch.cat([x, y]) for x, y in zip(kept[l][b], new)] if base[b] else new
        keep = [-1] * cap
        for b, path in enumerate(paths):
            keep[cu[b]:cu[b] + len(path)] = path
        n_keep.copy_(i32([len(p) for p in paths]))
        lead.keep_rows(plan, i32(keep), n_keep, lengths, layers=caches)
        lead.truncate(lengths)
        base = [b + len(p) for b, p in zip(base, paths)]
        assert lead.seqlens.tolist() == base == lengths.tolist()
        for l, c in enumerate(caches):
            for b in range(B):
                if base[b]:
                    assert all(torch.equal(x, y) for x, y in zip(rows(c, place(b, 0, base[b])), kept[l][b])), (round_, l, b)
        used = [p for b in range(B) for p in lead.page_table[b, :-(-base[b] // 128)].tolist()]
        free = lead.free[1:1 + int(lead.free[0])].tolist()
        assert sorted(used + free) == list(range(lead.n_pages))
    assert all(int(s.abs().sum()) == 0 for s in (plan.status, prompts.status, lead.status, *[w.status for w in spaces]))


@pytest.mark.parametrize("v_bits,chain", [(0, False), (3, False), (0, True)])
def test_a_whole_step_in_one_graph(v_bits, chain):
    """plan, write, attend, keep and truncate captured together and replayed with other drafts, lengths and paths: tables, pages and outputs are
    those of the calls made one by one."""
    pk = PhasorKey.from_spec(synth.make_layer("cfg2", 0, d_model=D, factor_gain=16.0))
    pk.set_second(0.002)
    B, cap, r = 3, 40, random.Random(21)
    g = torch.Generator(device="cuda").manual_seed(21)
    t = lambda *s: torch.randn(s, generator=g, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    n_new, parents, keep, n_keep = i32([0] * B), i32([-1] * cap), i32([-1] * cap), i32([0] * B)
    x, q, v = t(cap, D), 20 * t(cap, 32, 128), t(cap, 8, 128).to(torch.bfloat16)
    x0, v0 = t(400, D), t(400, 8, 128).to(torch.bfloat16)

    class One:
        def __init__(self):
            self.cache = pk.new_cache(B, 400, v_bits=v_bits)
            self.cache.use_page_pool()
            self.plan, self.ws = self.cache.step_plan(cap, tree=True), pk.tree_workspace(B, cap, 12, 400)
            self.scratch, self.lengths = pk.write_scratch(cap), i32([0] * B)
            self.out = torch.zeros((cap, 32, 128), dtype=torch.bfloat16, device="cuda")
            prompt = self.cache.step_plan(400)
            self.cache.plan_step(prompt, i32([130, 0, 250]))
            pk.write_paged(self.cache, x0, prompt.positions, prompt.slots, v=v0)

        def step(self):
            self.cache.plan_step(self.plan, n_new, parents=None if chain else parents)
            pk.write_paged(self.cache, x, self.plan.positions, self.plan.slots, v=v, scratch=self.scratch)
            pk.tree_step(self.cache, q, self.plan, self.ws, out=self.out)
            self.cache.keep_rows(self.plan, keep, n_keep, self.lengths)
            self.cache.truncate(self.lengths)

        def state(self):
            c, p = self.cache, self.plan
            return [c.page_table, c.seqlens, c.free, c.latent, c.vq if c.v_bits else c.v.view(torch.int16), p.cu, p.slots, p.mask, self.lengths, self.out]
    one, graphed = One(), One()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        graphed.step()
    for round_ in range(6):
        n = [r.choice([0, 1, 12, r.randint(0, 12)]) for _ in range(B)]
        ups = [[i - 1 if chain else r.randint(max(-1, i - 4), i - 1) for i in range(m)] for m in n]
        paths = []
        for up in ups:
            path = [r.randrange(len(up))] if up else []
            while path and up[path[0]] >= 0:
                path.insert(0, up[path[0]])
            paths.append(path)
        flat = lambda lists, pad: sum((l + [pad] * (m - len(l)) for l, m in zip(lists, n)), [])
        n_new.copy_(i32(n)), n_keep.copy_(i32([len(p) for p in paths]))
        parents[:sum(n)], keep[:sum(n)] = i32(flat(ups, -1)), i32(flat(paths, -1))
        for a in (x, v):
            a.copy_(t(*a.shape))
        q.copy_(20 * t(*q.shape))
        graph.replay()
        one.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(one.state(), graphed.state())), round_
    assert sum(one.cache.seqlens.tolist()) > 380
    assert all(int(s.abs().sum()) == 0 for o in (one, graphed) for s in (o.plan.status, o.cache.status, o.ws.status))
