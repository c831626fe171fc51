"""What the step's Python calls refuse or arrange before anything reaches a GPU: with stand-ins for the layer and its cache, on the CPU."""
import contextlib
import types

import pytest
import torch

from phasorkv_b200 import PagedLatentCache, PhasorKey, TreeWorkspace, _lib, build, patch
from phasorkv_b200.patch import LayerDecodeState


@pytest.fixture(scope="module", autouse=True)
def lib():
    build.build()


# ------------------------------------------------------------------------------------------------ verify
D, N_Q, N_KV = 32, 4, 2


class Recorder:
    """A layer and its cache that only note what is called, on which device."""

    def __init__(self, batch=2):
        self.calls, self.inside = [], None
        note = lambda name: lambda *a, **k: self.calls.append((name, self.inside))
        self.pk = types.SimpleNamespace(device=torch.device("cpu"), d_model=D, n_q=N_Q, n_kv=N_KV, head_dim=128, cache_width=64, write_paged=note("write"),
                                        write_scratch=lambda n: None, _tree_key=lambda: 0, tree_workspace=lambda *a, **k: types.SimpleNamespace(bytes=4, use=lambda b: None),
                                        tree_step=lambda cache, q, plan, ws, **k: (self.calls.append(("attend", self.inside)), torch.zeros(q.shape))[1])
        plan = types.SimpleNamespace(positions=None, slots=None)
        self.cache = types.SimpleNamespace(latent=torch.zeros(1), step_plan=lambda *a, **k: plan, plan_step=note("plan"), truncate=note("truncate"),
                                           keep_rows=note("keep"))
        st = self.state = object.__new__(LayerDecodeState)
        st.pk, st.cache, st.batch, st.max_tokens, st.lengths, st.drafted, st.tree = self.pk, self.cache, batch, 256, [5, 9], None, {}
        st.scratch = patch.VerifyScratch()

    @contextlib.contextmanager
    def on_device(self, device):
        self.inside = device
        yield 0
        self.inside = None


def tensors(B=2, n=3, **shapes):
    z = lambda name, *s: torch.zeros(shapes.get(name, s))
    return z("x", B, n, D), z("q", B, n, N_Q, 128), z("v", B, n, N_KV, 128)


@pytest.mark.parametrize("shapes", [dict(x=(2, 3, D // 2)), dict(x=(2, 3, 2 * D)), dict(q=(2, 3, N_Q // 2, 128)), dict(q=(2, 6, N_Q, 64)), dict(q=(3, 2, N_Q, 128)),
                                    dict(v=(2, 3, 2 * N_KV, 64)), dict(v=(3, 2, N_KV, 128)), dict(v=(2, 4, N_KV, 128))])
def test_verify_refuses_tensors_of_another_shape(shapes):
    """The write kernel reads d_model columns of every row: a narrower x would be read past its end."""
    r = Recorder()
    with pytest.raises(ValueError):
        r.state.verify(*tensors(**shapes))
    assert r.calls == [] and r.state.drafted is None


@pytest.mark.parametrize("which", [1, 2])
def test_verify_refuses_tensors_of_another_device(which):
    r, t = Recorder(), list(tensors())
    t[which] = t[which].to("meta")
    with pytest.raises(ValueError):
        r.state.verify(*t)
    assert r.calls == []


def test_verify_runs_on_the_device_of_its_cache(monkeypatch):
    """The writer's launches go to the current device: inside verify and accept that is the cache's, whatever the caller's is."""
    r = Recorder()
    monkeypatch.setattr(patch, "on_device", r.on_device, raising=False)
    r.state.verify(*tensors())
    r.state.accept([[0], [0, 1]])
    assert [c[0] for c in r.calls] == ["plan", "write", "attend", "keep", "truncate"]
    assert all(where == torch.device("cpu") for _, where in r.calls), r.calls


# ------------------------------------------------------------------------------------------------ accept in all layers
def two_layers(drafted):
    """A patch of two layers, of which those in `drafted` wait for accept."""
    p, rec = patch.PhasorKeyPatch(), [Recorder(), Recorder()]
    for i, r in enumerate(rec):
        if i in drafted:
            r.state.drafted = (types.SimpleNamespace(), [[-1, 0, 0], [-1, 0, 1]])
        p.states[i] = r.state
    return p, rec


@pytest.mark.parametrize("drafted,keep,error", [((0,), [[0], [0]], RuntimeError), ((0, 1), [[0], [1]], ValueError), ((0, 1), [[0]], ValueError)])
def test_accept_refuses_in_all_layers_or_none(drafted, keep, error):
    p, rec = two_layers(drafted)
    with pytest.raises(error):
        p.accept(keep)
    assert all(r.calls == [] and r.state.lengths == [5, 9] for r in rec)
    assert [r.state.drafted is not None for r in rec] == [i in drafted for i in range(2)]


def test_accept_refuses_a_path_that_one_layer_did_not_draft():
    p, rec = two_layers((0, 1))
    rec[1].state.drafted = (types.SimpleNamespace(), [[-1, -1, 0], [-1, 0, 1]])
    with pytest.raises(ValueError):
        p.accept([[0, 1], [0]])
    assert all(r.calls == [] and r.state.drafted is not None for r in rec)


def test_accept_takes_the_paths_from_an_iterator_once(monkeypatch):
    p, rec = two_layers((0, 1))
    monkeypatch.setattr(patch, "on_device", rec[0].on_device, raising=False)
    p.accept(iter(rows) for rows in ([0, 2], []))
    assert all([c[0] for c in r.calls] == ["keep", "truncate"] and r.state.lengths == [7, 9] and r.state.drafted is None for r in rec)


def test_dropping_all_drafts_ends_a_pass_that_failed_halfway(monkeypatch):
    p, rec = two_layers((0,))
    monkeypatch.setattr(patch, "on_device", rec[0].on_device, raising=False)
    p.accept([[], []])
    assert [[c[0] for c in r.calls] for r in rec] == [["keep", "truncate"], []]
    assert all(r.state.lengths == [5, 9] and r.state.drafted is None for r in rec)
    with pytest.raises(RuntimeError):
        p.accept([[], []])


# ------------------------------------------------------------------------------------------------ page pool and sharing
def caches(k):
    return [PagedLatentCache(256, 8, 128, 2, 512, "cpu") for _ in range(k)]


@pytest.mark.parametrize("who", [0, 1, 2])
def test_a_page_pool_made_after_sharing_is_everyones(who):
    a, b, c = caches(3)
    b.share_pages(a), c.share_pages(b)
    (a, b, c)[who].use_page_pool()
    assert a.free is b.free is c.free and a.free.tolist() == [8, 7, 6, 5, 4, 3, 2, 1, 0] and int(a.page_table.max()) == -1


def test_a_page_pool_is_refilled_in_place():
    """A captured step and the caches that share the pool go on with the same array."""
    a, b = caches(2)
    a.use_page_pool()
    b.share_pages(a)
    pool = a.free
    pool[0] = 3
    a.page_table[0, 0], a.seqlens[1] = 4, 77
    b.use_page_pool()
    assert a.free is pool and b.free is pool and pool.tolist() == [8, 7, 6, 5, 4, 3, 2, 1, 0]
    assert int(a.page_table.max()) == -1 and a.seqlens.tolist() == [0, 0]


def test_a_cache_that_shares_with_another_leaves_its_first_owner():
    a, b, c = caches(3)
    b.share_pages(a)
    b.share_pages(c)
    a.use_page_pool()
    assert b.free is None and c.free is None and b.page_table is c.page_table
    c.use_page_pool()
    assert b.free is c.free and b.free is not a.free
    c.share_pages(c)
    assert c.free is b.free


# ------------------------------------------------------------------------------------------------ devices of a tree step
@pytest.mark.parametrize("wrong", ["workspace", "layer"])
def test_tree_step_refuses_another_devices_workspace_or_layer(wrong):
    cpu = torch.zeros(1)
    pk = PhasorKey.from_factors(torch.zeros((8, 128), dtype=torch.complex64), torch.zeros((128, 16), dtype=torch.complex64), torch.arange(128) // 2, 32, 8, 128,
                                torch.ones(64, dtype=torch.float64), device="cpu")
    pk._dev = {"Bw": cpu.to("meta") if wrong == "layer" else cpu, "layer": _lib.Layer()}
    cache = PagedLatentCache(256, 8, 128, 1, 128, "cpu")
    ws = object.__new__(TreeWorkspace)
    ws.buffer = ws.status = cpu.to("meta") if wrong == "workspace" else cpu
    ws.batch, ws.capacity, ws.max_draft, ws.max_pages, ws.key, ws.at, ws.bytes, ws.status_at = 1, 4, 4, 1, pk._tree_key(), 0, 0, 0
    with pytest.raises(ValueError, match="device"):
        pk.tree_step(cache, torch.zeros((4, 32, 128)), cache.step_plan(4), ws)


def test_a_workspace_refuses_a_buffer_that_does_not_hold_it():
    ws = object.__new__(TreeWorkspace)
    ws.bytes = 2048
    room = torch.zeros(8192, dtype=torch.uint8)
    at = -room.data_ptr() % 1024
    for bad in (room[at:at + 2047], room[at + 16:at + 4096], room[at:at + 4096].view(torch.int32), room[at:at + 4096 + 2048:2]):
        with pytest.raises(ValueError):
            ws.use(bad)
    ws.use(room[at:at + 2048])
    assert ws.at == room.data_ptr() + at
