"""Attention of drafted trees over the paged latent cache: refusals on the CPU, and on the GPU the outputs against the
formula in 64 bits on what the pages hold.

Tolerances. The result carries three roundings to bf16 of at most 2^-8 of a value: of the weights, in numerator and in
denominator (2 x 2^-8 A with A = sum p |v|), and of the output (2^-8 |O| <= 2^-8 A). The query's four NVFP4 terms leave
7e-5 of a logit; the logits here stay below 25, so a weight is off by at most e^(2 x 1.75e-3) - 1 < 2^-8. Together:
|error| <= 4 x 2^-8 A for every value. In the 2-norm the two independent roundings are uniform over a half step, 2^-8 / sqrt(3)
each, 3.2e-3 together, and the logits' share 7e-5 x |S| adds less than 1.75e-3: 5e-3."""
import ctypes
import random

import pytest
import torch

from phasorkv_b200 import PagedLatentCache, PhasorKey, _lib, build, synth

PAGE = 128
ELEM, NORM = 4 * 2.0 ** -8, 5e-3


def layer(n_q, n_kv, layout="freq2", seed=0, **kw):
    """Factors of any head layout; `layout` as in the package's configurations."""
    R, R_s, n_slow = {"freq2": (128, 0, 0), "band8": (120, 16, 8), "freq1": (64, 0, 0), "odd": (52, 8, 3)}[layout]
    g = torch.Generator().manual_seed(seed)
    c = lambda *s: torch.complex(torch.randn(s, generator=g), torch.randn(s, generator=g)) * 0.7071
    freq = (torch.arange(R) * (64 - n_slow)) // R
    return PhasorKey.from_factors(c(n_kv, R), torch.zeros((R, 16), dtype=torch.complex64), freq, n_q, n_kv, 128, synth.rope_inv_freq(128, 5e5),
                                  torch.randn((n_kv, 2 * n_slow, R_s), generator=g) * 0.3 if R_s else None,
                                  torch.zeros((R_s, 16)) if R_s else None, torch.arange(64 - n_slow, 64), **kw)


def tree_words(r, n, kind):
    words = []
    for i in range(n):
        up = i - 1 if kind == "chain" else r.randint(max(-1, i - 6), i - 1)
        words.append({"any": lambda: r.choice([0, r.getrandbits(64), (1 << 64) - 1, 1 << i]), "none": lambda: 0}.get(
            kind, lambda: (words[up] if up >= 0 else 0) | 1 << i)())
    return [w - (1 << 64) if w >> 63 else w for w in words]


class Case:
    """A batch with `base` cached and `n` drafted tokens a sequence, its pages scattered over the pool."""

    def __init__(self, pk, base, n, mask="tree", v_bits=0, q_dtype=torch.bfloat16, seed=3, spare=2, first_page=0, pad=0):
        self.pk, self.base, self.n, r = pk, base, n, random.Random(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        B, W = len(base), pk.cache_width
        most = max(1, max(b + m for b, m in zip(base, n)))
        pages = -(-most // PAGE)
        pk.set_second(0.02)
        self.cache = cache = PagedLatentCache(W, pk.n_kv, 128, B, most, "cuda", n_pages=first_page + B * pages + spare, v_bits=v_bits)
        order = torch.randperm(cache.n_pages - first_page, generator=g, device="cuda")[:B * pages] + first_page
        cache.page_table.copy_(order.view(B, pages))
        slots = (cache.page_table.reshape(-1, 1) * PAGE + torch.arange(PAGE, device="cuda", dtype=torch.int32)).reshape(-1).to(torch.int32)
        sigma = torch.linspace(2.5, 0.5, W, device="cuda")
        cache.quantize_rows(torch.randn((len(slots), W), generator=g, device="cuda") * sigma, slots, pk.second)
        cache.write_v(torch.randn((len(slots), pk.n_kv, 128), generator=g, device="cuda").to(torch.bfloat16), slots)
        cache.seqlens.copy_(torch.tensor([b + m for b, m in zip(base, n)], dtype=torch.int32))
        N = sum(n)
        self.cap = N + pad
        self.words = [tree_words(r, m, mask) if mask else [(2 << i) - 1 if i < 62 else (-1 if i == 63 else (1 << 63) - 1) for i in range(m)] for m in n]
        self.positions = [[b + r.randint(0, i) for i in range(m)] for b, m in zip(base, n)]
        self.plan = plan = cache.step_plan(self.cap, tree=bool(mask))
        plan.cu.copy_(torch.tensor([sum(n[:b]) for b in range(B + 1)], dtype=torch.int32))
        plan.positions[:N] = torch.tensor(sum(self.positions, []), dtype=torch.int32)
        if mask:
            plan.mask[:N] = torch.tensor(sum(self.words, []), dtype=torch.int64)
        self.q = torch.randn((self.cap, pk.n_q, 128), generator=g, device="cuda").to(q_dtype)
        self.max_draft = max(1, max(n))
        self.ws = pk.tree_workspace(B, self.cap, self.max_draft, cache.max_pages * PAGE)

    def slots(self, b, lo, hi):
        t = torch.arange(lo, hi, device="cuda", dtype=torch.int32)
        return self.cache.slots(torch.full_like(t, b), t)

    def run(self, **kw):
        return self.pk.tree_step(self.cache, self.q, self.plan, self.ws, **kw)

    def formula(self, b, most=25):
        """(O, A = sum p |v|) of sequence b in doubles, on what the pages hold."""
        pk, base, n = self.pk, self.base[b], self.n[b]
        lo = sum(self.n[:b])
        rep, R, dev = pk.n_q // pk.n_kv, pk.R, "cuda"
        slots = self.slots(b, 0, base + n)
        C = self.cache.read(slots, pk.second, codes=False)[0].double()
        V = self.cache.v_rows(slots).double()
        q = self.q[lo:lo + n].double()
        ang = torch.tensor(self.positions[b], dtype=torch.float64, device=dev)[:, None] * pk.inv_freq.to(dev)
        cs, sn = ang.cos()[:, None], ang.sin()[:, None]
        x, y, f = q[..., :64], q[..., 64:], pk.freq.to(dev)
        zr, zi = (x * cs - y * sn)[..., f], (x * sn + y * cs)[..., f]
        see = torch.ones((n, base + n), dtype=torch.bool)
        for i in range(n):
            for j in range(n):
                see[i, base + j] = bool(self.words[b][i] >> j & 1)
        see = see.to(dev)
        O, A = (torch.zeros((n, pk.n_q, 128), dtype=torch.float64, device=dev) for _ in range(2))
        for g in range(pk.n_kv):
            h = slice(g * rep, (g + 1) * rep)
            ar, ai = pk.A[g].real.double().to(dev), pk.A[g].imag.double().to(dev)
            qa = [ar * zr[:, h] + ai * zi[:, h], ar * zi[:, h] - ai * zr[:, h]]
            if pk.R_s:
                s = pk.slow.to(dev)
                qa.append(torch.cat([x[:, h][..., s], y[:, h][..., s]], -1) @ pk.A_s[g].double().to(dev))
            S = torch.cat(qa, -1) @ C.T * 128 ** -0.5
            S = torch.where(see[:, None], S, -torch.inf)
            assert not (S[torch.isfinite(S)].abs() >= most).any()               # what the tolerance counts on
            P = torch.softmax(S, -1)
            P = torch.where(see.any(-1)[:, None, None], P, torch.zeros_like(P))
            for i in range(n):                                                  # only what a row sees enters its sums
                v = V[see[i], g]
                O[i, h], A[i, h] = P[i][:, see[i]] @ v, P[i][:, see[i]] @ v.abs()
        return O, A

    def check(self, out, skip=()):
        torch.cuda.synchronize()
        assert int(self.ws.status.abs().sum()) == 0, self.ws.status.tolist()
        for b in range(len(self.base)):
            lo, n = sum(self.n[:b]), self.n[b]
            if n == 0:
                continue
            O, A = self.formula(b)
            got = out[lo:lo + n].double()
            rows = [i for i in range(n) if (b, i) not in skip]
            d = (got - O)[rows]
            assert not d.isnan().any(), (b, d.isnan().nonzero()[:4])
            assert (d.abs() <= ELEM * A[rows]).all(), (b, float((d.abs() / A[rows].clamp_min(1e-30)).max()))
            assert float(d.norm()) <= NORM * float(O[rows].norm()), (b, float(d.norm() / O[rows].norm()))


# ------------------------------------------------------------------------------------------------ refusals (no GPU)
@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def c_layer(**k):
    d = dict(d_model=16, n_q=32, n_kv=8, head_dim=128, R=128, R_s=0, n_slow=0, attn_scale=1.0, second=1.0)
    d.update(k)
    return _lib.Layer(*[d[n] for n in ("d_model", "n_q", "n_kv", "head_dim", "R", "R_s", "n_slow", "attn_scale", "second")],
                      4096, 4096, 4096, 4096, 4096, 4096, 4096, 0, 0)


def test_c_entry_refuses_bad_arguments(lib):
    L, C, pg = c_layer(), _lib.Cache(4096, 4096, 8, 256, 8, 128), _lib.Pages(4096, 4096, 0, 2, 4, 8)
    size = lib.pkv_tree_workspace_bytes(ctypes.byref(L), 2, 8, 4)
    assert size > 0 or size == 0
    assert lib.pkv_tree_workspace_bytes(None, 2, 8, 4) == -1 and lib.pkv_tree_workspace_bytes(ctypes.byref(L), -1, 8, 4) == -1
    assert lib.pkv_tree_workspace_bytes(ctypes.byref(L), 2, 0, 4) == -1 and lib.pkv_tree_workspace_bytes(ctypes.byref(L), 2, 65, 4) == -2

    def call(L=L, C=C, pg=pg, q=4096, dt=1, pos=4096, cu=4096, n=4, md=8, ws=4096, wb=None, out=4096):
        return lib.pkv_tree_attn(ctypes.byref(L) if L else None, ctypes.byref(C) if C else None, ctypes.byref(pg) if pg else None, q, dt, pos, None,
                                 cu, n, md, ws, size if wb is None else wb, out, None, None)
    assert call(L=None) == -1 and call(C=None) == -1 and call(pg=None) == -1
    assert call(q=None) == -1 and call(pos=None) == -1 and call(cu=None) == -1 and call(out=None) == -1
    assert call(q=4104) == -1 and call(out=4098) == -1                          # misaligned
    assert call(n=-1) == -1 and call(md=0) == -1 and call(md=65) == -2 and call(dt=2) == -2
    assert call(L=c_layer(head_dim=64), C=_lib.Cache(4096, 4096, 8, 256, 8, 64)) == -2
    assert call(L=c_layer(n_q=65, n_kv=1), C=_lib.Cache(4096, 4096, 8, 256, 1, 128)) == -2
    assert call(C=_lib.Cache(4096, 4096, 8, 128, 8, 128)) == -1                 # another latent width
    assert call(C=_lib.Cache(4096, 4096, 8, 256, 4, 128)) == -1                 # other kv heads
    assert call(C=_lib.Cache(4096, 0, 8, 256, 8, 128)) == -1                    # no values
    assert call(C=_lib.Cache(4096, 0, 8, 256, 8, 128, 0, 3)) == -1              # no quantised values
    assert call(pg=_lib.Pages(4096, 4096, 0, -1, 4, 8)) == -1 and call(pg=_lib.Pages(4096, 4096, 0, 4097, 4, 8)) == -2
    assert call(pg=_lib.Pages(4096, 4096, 0, 0, 4, 8)) == 0 and call(n=0) == 0  # nothing to do


def test_no_cpu_path():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    with pytest.raises(_lib.PhasorKVError):
        layer(32, 8, device="cpu").tree_workspace(1, 4, 4, 128)


# ------------------------------------------------------------------------------------------------ on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("n_q,n_kv,layout", [(32, 8, "freq2"), (32, 4, "freq2"), (32, 32, "freq1"), (16, 8, "band8"), (24, 8, "freq2"),
                                             (64, 8, "freq1"), (28, 4, "band8"), (7, 7, "odd"), (64, 1, "freq2"), (40, 8, "freq1")])
@pytest.mark.parametrize("v_bits", [0, 3, 2])
def test_head_layouts(n_q, n_kv, layout, v_bits):
    c = Case(layer(n_q, n_kv, layout), [300, 0, 127, 129, 640], [5, 3, 0, 17, 1], v_bits=v_bits)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("base,n", [([0], [1]), ([1], [1]), ([0, 0], [64, 2]), ([127], [1]), ([128], [1]), ([126], [2]), ([127, 128, 129], [64, 64, 64]),
                                    ([256, 255], [33, 32]), ([1000, 5, 0], [7, 0, 9]), ([0, 0, 0], [0, 0, 1]), ([4095], [64]), ([5000, 300], [16, 8])])
@pytest.mark.parametrize("mask", ["tree", "any", None])
def test_lengths_and_masks(base, n, mask):
    c = Case(layer(32, 8), base, n, mask=mask, seed=len(base) + sum(n))
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 9, 12, 16, 17, 31, 32, 33, 48, 63, 64])
@pytest.mark.parametrize("n_q,n_kv,layout,v_bits", [(32, 8, "freq2", 0), (32, 32, "freq1", 0), (32, 8, "freq2", 3)])
def test_every_tile_shape(n, n_q, n_kv, layout, v_bits):
    c = Case(layer(n_q, n_kv, layout), [391, 77], [n, max(0, n - 3)], v_bits=v_bits, q_dtype=torch.float32)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("B,v_bits", [(40, 0), (300, 0), (70, 3)])
def test_ragged_batches(B, v_bits):
    r = random.Random(B)
    base = [r.choice([0, 1, r.randint(0, 900)]) for _ in range(B)]
    c = Case(layer(32, 8), base, [r.choice([0, 1, r.randint(0, 20)]) for _ in range(B)], v_bits=v_bits)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("base,n,v_bits", [(40000, 6, 0), (70001, 40, 0), (50000, 9, 3)])
def test_long_sequences(base, n, v_bits):
    c = Case(layer(32, 8), [base, 17], [n, 2], v_bits=v_bits)
    c.check(c.run())


@pytest.mark.gpu
def test_rows_that_see_nothing_are_zero():
    c = Case(layer(32, 8), [0, 200], [9, 4], mask="none")
    out = c.run(out=torch.full(c.q.shape, 7.0, device="cuda", dtype=torch.bfloat16))
    assert float(out[:9].abs().max()) == 0.0
    c.check(out)


@pytest.mark.gpu
@pytest.mark.parametrize("v_bits", [0, 3])
def test_rows_behind_the_last_sequence_stay(v_bits):
    c = Case(layer(32, 8), [140, 3], [4, 2], v_bits=v_bits, pad=5)
    out = torch.full(c.q.shape, 7.0, device="cuda", dtype=torch.bfloat16)
    assert c.run(out=out) is out
    c.check(out)
    assert (out[6:] == 7).all()


def poison(c, slots, kind):
    """Infinities and NaN in the stored values of `slots`, NaN in their latent scales (bit pattern 0x7F) if asked."""
    cache = c.cache
    s = slots.long()
    page, row = s // PAGE, s % PAGE
    bad = {"nan": float("nan"), "inf": float("inf"), "-inf": float("-inf")}[kind]
    if cache.v_bits:
        per = cache.n_kv * 8448
        pool = cache.vq.view(-1, per)
        for g in range(cache.n_kv):
            at = cache.n_kv * 8192 + g * 256 + row * 2
            b16 = torch.tensor([bad], dtype=torch.bfloat16).view(torch.uint8).tolist()
            pool[page, at], pool[page, at + 1] = b16[0], b16[1]
    else:
        cache.v[page, :, row, :] = bad
    Wp = 128 if cache.W <= 128 else 256
    lat = cache.latent.view(-1, cache.page_bytes)
    for j in range(Wp // 16):
        lat[page, PAGE * Wp // 2 + (j // 4) * 512 + (row % 32) * 16 + (row // 32) * 4 + j % 4] = 0x7F


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("base,n,v_bits", [(200, 9, 0), (120, 30, 0), (0, 64, 0), (383, 2, 0), (200, 9, 3), (120, 30, 2)])
def test_masked_rows_may_hold_anything(kind, base, n, v_bits):
    """Two branches: the rows of one hold infinities and NaN, and so does everything behind the sequence in its last page. Who does
    not see them is not touched by them, who does gets NaN."""
    c = Case(layer(32, 8), [base, 40], [n, 3], mask="chain", v_bits=v_bits)
    half = n // 2
    good = sum(1 << i for i in range(half))                                     # rows 0 .. half-1: one branch; the rest another
    words = [w & good if i < half else (w & ~good) for i, w in enumerate(c.words[0])]
    c.words[0] = [w - (1 << 64) if w >> 63 & 1 and w > 0 else w for w in words]
    c.plan.mask[:n] = torch.tensor(c.words[0], dtype=torch.int64)
    end = -(-(base + n) // PAGE) * PAGE
    poison(c, c.slots(0, base + n, end), kind) if end > base + n else None
    poison(c, c.slots(0, base + half, base + half + 1), kind)                   # the root of the second branch
    out = c.run()
    c.check(out, skip={(0, i) for i in range(half, n)})
    assert out[half:n].isnan().all()


@pytest.mark.gpu
def test_nan_among_the_cached_rows_reaches_every_output():
    c = Case(layer(32, 8), [300], [3])
    s = c.slots(0, 20, 21).long()
    c.cache.v[s // PAGE, 2, s % PAGE, 5] = float("nan")
    out = c.run()
    assert out[:, 8:12, 5].isnan().all()
    out[:, 8:12, 5] = 0
    assert not out.isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
def test_bad_pages_are_reported_not_read(bad):
    c = Case(layer(32, 8), [300, 400], [3, 2])
    c.cache.page_table[0, 1] = bad
    c.run()
    torch.cuda.synchronize()
    assert int(c.ws.status[0]) == 2


@pytest.mark.gpu
def test_sequences_out_of_range_are_left_out():
    c = Case(layer(32, 8), [300, 400, 20], [3, 9, 2])
    ws = c.pk.tree_workspace(3, c.cap, 8, 512)                                  # the second sequence has nine rows
    out = torch.full(c.q.shape, 7.0, device="cuda", dtype=torch.bfloat16)
    c.pk.tree_step(c.cache, c.q, c.plan, ws, out)
    assert ws.status[:2].tolist() == [4, 1] and (out[3:12] == 7).all()
    O, A = c.formula(2)
    assert ((out[12:].double() - O).abs() <= ELEM * A).all()
    c.cache.seqlens[0] = 2                                                      # fewer tokens than drafted
    ws.status.zero_()
    out.fill_(7.0)
    c.pk.tree_step(c.cache, c.q, c.plan, c.ws, out)
    assert c.ws.status[:2].tolist() == [4, 0] and (out[:3] == 7).all() and not (out[3:] == 7).all(-1).any()


@pytest.mark.gpu
def test_python_call_refuses_what_it_cannot_read():
    c = Case(layer(32, 8), [30], [4])
    pk, q = c.pk, c.q
    for bad in (q.half(), q[:, :16], q.transpose(0, 1).contiguous().transpose(0, 1), q.cpu(), torch.cat([q, q])):
        with pytest.raises(ValueError):
            pk.tree_step(c.cache, bad, c.plan, c.ws)
    with pytest.raises(ValueError):
        pk.tree_step(c.cache, q, c.plan, c.ws, out=torch.empty_like(q, dtype=torch.float32))
    with pytest.raises(ValueError):
        pk.tree_step(c.cache, q, c.plan, pk.tree_workspace(2, 4, 4, 128))       # another batch
    with pytest.raises(ValueError):
        pk.tree_step(c.cache, q, c.plan, layer(32, 4).tree_workspace(1, 4, 4, 128))
    for args in ((1, 4, 0, 128), (1, 4, 65, 128), (1, -1, 4, 128), (1, 4, 4, 0)):
        with pytest.raises(ValueError):
            pk.tree_workspace(*args)
    with pytest.raises(_lib.PhasorKVError):
        other = PagedLatentCache(128, 8, 128, 1, 128, "cuda")                   # another latent width
        pk.tree_step(other, q, c.plan, c.ws)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Pages behind the first 4 GB of the value pool."""
    c = Case(layer(32, 8), [700, 100], [6, 3], first_page=17000)
    assert c.cache.v.numel() * 2 > 1 << 32
    c.check(c.run())


@pytest.mark.gpu
def test_captured_step_follows_the_lengths():
    """One captured launch sequence serves steps of other lengths, masks and pages, and gives the eager call's bits."""
    c = Case(layer(32, 8), [900, 300, 77], [9, 16, 4], pad=40)
    out = torch.zeros(c.q.shape, device="cuda", dtype=torch.bfloat16)
    c.ws = c.pk.tree_workspace(3, c.cap, 32, c.cache.max_pages * PAGE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.run(out=out)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        c.run(out=out)
    for base, n in ([900, 300, 77], [9, 16, 4]), ([3, 640, 0], [1, 0, 31]), ([877, 0, 900], [32, 2, 9]):
        r = random.Random(sum(n))
        c.base, c.n = base, n
        c.words = [tree_words(r, m, "tree") for m in n]
        c.positions = [[b + i // 2 for i in range(m)] for b, m in zip(base, n)]
        N = sum(n)
        c.plan.cu.copy_(torch.tensor([sum(n[:b]) for b in range(4)], dtype=torch.int32))
        c.plan.positions[:N] = torch.tensor(sum(c.positions, []), dtype=torch.int32)
        c.plan.mask[:N] = torch.tensor(sum(c.words, []), dtype=torch.int64)
        c.cache.seqlens.copy_(torch.tensor([b + m for b, m in zip(base, n)], dtype=torch.int32))
        g.replay()
        c.check(out)
        assert torch.equal(out[:N], c.run()[:N])


@pytest.mark.gpu
def test_two_calls_at_once_and_the_same_bits_again():
    a, b = Case(layer(32, 8), [3000, 500], [12, 7]), Case(layer(32, 32, "freq1"), [2000], [20], v_bits=3, seed=9)
    want = a.run(), b.run()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s1):
            x = a.run()
        with torch.cuda.stream(s2):
            y = b.run()
        torch.cuda.synchronize()
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])
    a.check(want[0]), b.check(want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
def test_a_query_that_is_not_finite_makes_its_rows_nan(bad):
    c = Case(layer(32, 8), [700, 90], [9, 4], q_dtype=torch.float32)
    want = c.run()
    c.q[3, 17, 40] = float(bad)
    out = c.run()
    assert out[3, 17].isnan().all()
    out[3, 17] = want[3, 17]
    assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("v_bits", [0, 2])
def test_peaked_logits(v_bits):
    """Queries 12 times as large: one token has most of the weight. The query's terms leave 7e-5 of a logit, here at most 300, so
    a weight is off by e^(2 x 0.021) - 1 = 0.043 of itself at most and the result by as much of A, next to the roundings."""
    c = Case(layer(32, 8), [900, 130], [11, 40], v_bits=v_bits, q_dtype=torch.float32)
    c.q *= 12.0
    out = c.run()
    torch.cuda.synchronize()
    for b, (lo, n) in enumerate(((0, 11), (11, 40))):
        O, A = c.formula(b, most=300)
        assert ((out[lo:lo + n].double() - O).abs() <= (ELEM + 0.043) * A).all()


@pytest.mark.gpu
def test_no_sequence_has_a_draft():
    c = Case(layer(32, 8), [300, 0], [0, 0], pad=3)
    out = torch.full(c.q.shape, 7.0, device="cuda", dtype=torch.bfloat16)
    c.run(out=out)
    torch.cuda.synchronize()
    assert (out == 7).all() and int(c.ws.status.abs().sum()) == 0


@pytest.mark.gpu
def test_result_in_place_of_the_queries():
    c = Case(layer(32, 8), [2900, 130], [30, 7])
    want = c.run()
    assert torch.equal(c.run(out=c.q), want)


@pytest.mark.gpu
def test_many_sequences():
    r = random.Random(1)
    base = [r.choice([0, 5, 126, 128, 200]) for _ in range(1500)]
    c = Case(layer(32, 4), base, [r.choice([0, 1, 2, 9]) for _ in base])
    c.check(c.run())


@pytest.mark.gpu
def test_captured_graphs_share_a_workspace():
    """Two layers' steps captured on their own with one workspace, replayed in any order on one stream."""
    a, b = Case(layer(32, 8), [900, 31], [9, 16]), Case(layer(32, 8, seed=4), [500, 800], [9, 16], seed=8)
    b.ws = a.ws = a.pk.tree_workspace(2, a.cap, 16, 1024)
    outs, graphs = [], []
    for c in (a, b):
        out = torch.zeros(c.q.shape, device="cuda", dtype=torch.bfloat16)
        c.run(out=out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run(out=out)
        outs.append(out)
        graphs.append(g)
    for i in (0, 1, 1, 0, 0, 1, 0):
        outs[i].zero_()
        graphs[i].replay()
        (a, b)[i].check(outs[i])


@pytest.mark.gpu
@pytest.mark.parametrize("n_q,n_kv,layout", [(64, 8, "freq1"), (64, 1, "freq2"), (64, 32, "freq1"), (48, 16, "band8")])
@pytest.mark.parametrize("base,n", [([700, 5, 2100], [64, 64, 64]), ([700, 5, 2100], [64, 1, 33])])
def test_more_tiles_than_a_gang_has_ctas(n_q, n_kv, layout, base, n):
    """Several passes over a sequence's pages, all sequences alike and not."""
    c = Case(layer(n_q, n_kv, layout), base, n)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("v_bits", [0, 3])
def test_a_reference_that_moves_on_every_page(v_bits):
    """Cached rows that grow from page to page: every page's maximum passes the row's reference, sums and results are rescaled."""
    c = Case(layer(32, 8), [1400, 600], [20, 3], v_bits=v_bits, q_dtype=torch.float32)
    W, most = c.pk.cache_width, 0.0
    for b, T in enumerate((1420, 603)):
        s = c.slots(b, 0, T)
        grow = (torch.arange(T, device="cuda") // PAGE + 1)[:, None] / (T // PAGE + 1.0)
        g = torch.Generator(device="cuda").manual_seed(b)
        c.cache.quantize_rows(torch.randn((T, W), generator=g, device="cuda") * grow * torch.linspace(2.5, 0.5, W, device="cuda"), s, c.pk.second)
    c.q *= 8.0
    out = c.run()
    torch.cuda.synchronize()
    for b, (lo, n) in enumerate(((0, 20), (20, 3))):                    # logits up to 300: as with peaked logits
        O, A = c.formula(b, most=300)
        assert ((out[lo:lo + n].double() - O).abs() <= (ELEM + 0.043) * A).all()


@pytest.mark.gpu
@pytest.mark.parametrize("v_bits", [0, 3])
def test_a_chain_planned_where_a_tree_was(v_bits):
    """One plan with masks serves a step of a tree and, planned again without parents, a chain."""
    base, n = [300, 64, 127], [9, 5, 12]
    c = Case(layer(32, 8), base, n, mask="any", v_bits=v_bits)
    c.check(c.run())
    c.cache.seqlens.copy_(torch.tensor(base, dtype=torch.int32))
    c.cache.plan_step(c.plan, torch.tensor(n, dtype=torch.int32, device="cuda"))
    c.words = [tree_words(random.Random(0), m, "chain") for m in n]
    c.positions = [[b + i for i in range(m)] for b, m in zip(base, n)]
    c.check(c.run())


@pytest.mark.gpu
def test_the_status_words_of_a_tree_step_belong_together():
    """A sequence that is left out (noticed by the operand launch) and a bad page (by the attention): one of the two, not a mixture."""
    c = Case(layer(32, 8), [700, 400, 20], [3, 9, 2])
    ws = c.pk.tree_workspace(3, c.cap, 8, c.cache.max_pages * PAGE)
    c.cache.page_table[0, 2] = -1
    for _ in range(20):
        ws.status.zero_()
        c.pk.tree_step(c.cache, c.q, c.plan, ws)
        assert ws.status[:2].tolist() in ([4, 1], [2, 2])
    ws.status.copy_(torch.tensor([4, 77, 0, 0], dtype=torch.int32))               # not cleared: the first problem stays
    c.pk.tree_step(c.cache, c.q, c.plan, ws)
    assert ws.status[:2].tolist() == [4, 77]


# The kernel's own roundings, counted one by one (the limits above leave room for one more that it no longer has): a weight is rounded to
# bf16 once, in the numerator alone (2^-8 A), the result once (2^-8 |O|); the sum takes the weights themselves. The cubic that forms a part of
# the weights is off by 7.5e-5 of them, in numerator and denominator. An NVFP4 term leaves 0.092 to 0.095 of what it is formed from
# (2-norm, of normal columns; E2M1 with a scale per 16 of them): 7.8e-4 after three terms, 7.2e-5 after four, here 0.096^4; a logit is off by TERMS s, s = (sum q'_k^2 c_k^2 / d)^1/2,
# in the 2-norm over many of them, since the residuals' signs are independent of the row. A single one stays below five times that.
# Uniform over a half step, a rounding is 2^-8 / 3^1/2 of the value in the 2-norm.
TERMS, ONE = 8.5e-5, 2.0 ** -8 / 3 ** 0.5


def spread(c, b, see):
    """(P, s, V) of sequence b: weights [n, H, T] and logit scales in doubles, values of each query head [H, T, d]."""
    pk, n, base = c.pk, c.n[b], c.base[b]
    lo, rep, dev = sum(c.n[:b]), pk.n_q // pk.n_kv, "cuda"
    slots = c.slots(b, 0, base + n)
    C, V = c.cache.read(slots, pk.second, codes=False)[0].double(), c.cache.v_rows(slots).double()
    q = c.q[lo:lo + n].double()
    ang = torch.tensor(c.positions[b], dtype=torch.float64, device=dev)[:, None] * pk.inv_freq.to(dev)
    z = (torch.complex(q[..., :64], q[..., 64:]) * torch.polar(torch.ones_like(ang), ang)[:, None])[..., pk.freq.to(dev)]
    z = pk.A.to(torch.complex128).to(dev).conj().repeat_interleave(rep, 0)[None] * z
    qa = torch.cat([z.real, z.imag], -1)
    S = torch.where(see[:, None], qa @ C.T * 128 ** -0.5, -torch.inf)
    return torch.softmax(S, -1), (qa ** 2 @ C.T ** 2 / 128).sqrt(), V.permute(1, 0, 2).repeat_interleave(rep, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("n_q,n_kv,layout,v_bits,n", [(32, 8, "freq2", 0, 16), (32, 8, "freq2", 0, 64), (32, 32, "freq1", 0, 8), (32, 8, "freq2", 3, 12)])
def test_no_more_roundings_than_counted(n_q, n_kv, layout, v_bits, n):
    c = Case(layer(n_q, n_kv, layout), [1900], [n], mask="chain", v_bits=v_bits, q_dtype=torch.float32)
    out = c.run().double()
    see = torch.ones((n, 1900 + n), dtype=torch.bool, device="cuda").tril(1900)
    P, s, V = spread(c, 0, see)
    O, A = c.formula(0)
    Q2 = torch.einsum("nht,htd->nhd", P ** 2, V ** 2)                             # what independent errors of the weights add up to, squared
    L2 = torch.einsum("nht,htd->nhd", (P * s) ** 2, V ** 2) + torch.einsum("nht,nhd->nhd", (P * s) ** 2, O ** 2)
    most = 5 * TERMS * torch.where(see[:, None], s, 0.0).amax()
    assert ((out - O).abs() <= 2.0 ** -8 * O.abs() + (2.0 ** -8 + 4 * 7.5e-5 + 2 * most) * A).all()
    limit = (ONE ** 2 * (Q2.sum() + (O ** 2).sum()) + TERMS ** 2 * L2.sum()).sqrt() + 2 * 7.5e-5 * O.norm()
    assert float((out - O).norm()) <= float(limit), (float((out - O).norm() / O.norm()), float(limit / O.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("n_q,n_kv,layout", [(32, 8, "freq2"), (32, 32, "freq1")])
def test_all_four_terms_of_the_query_count(n_q, n_kv, layout):
    """Rows that see two drafted tokens of nearly the same large logit: the difference of the logits' errors decides, and three terms would leave
    ten times as much. Queries 60 times as large; for each row the pair of head 0 whose logits are closest."""
    n = 64
    c = Case(layer(n_q, n_kv, layout), [0], [n], mask="chain", q_dtype=torch.float32)
    c.q *= 60.0
    everything = torch.ones((n, n), dtype=torch.bool, device="cuda")
    pk = c.pk
    q = c.q.double()
    ang = torch.tensor(c.positions[0], dtype=torch.float64, device="cuda")[:, None] * pk.inv_freq.to("cuda")
    z = (torch.complex(q[:, 0, :64], q[:, 0, 64:]) * torch.polar(torch.ones_like(ang), ang))[:, pk.freq.to("cuda")] * pk.A[0].to(torch.complex128).to("cuda").conj()
    S = torch.cat([z.real, z.imag], -1) @ c.cache.read(c.slots(0, 0, n), pk.second, codes=False)[0].double().T * 128 ** -0.5
    value, order = S.sort(-1)
    near = (value[:, 1:] - value[:, :-1]).argmin(-1)
    pairs = torch.stack([order.gather(1, near[:, None]), order.gather(1, near[:, None] + 1)], -1)[:, 0].tolist()
    words = [1 << j | 1 << k for j, k in pairs]
    c.words = [[w - (1 << 64) if w >> 63 else w for w in words]]
    c.plan.mask[:n] = torch.tensor(c.words[0], dtype=torch.int64)
    out = c.run().double()[:, 0]
    see = torch.zeros_like(everything)
    for i, (j, k) in enumerate(pairs):
        see[i, j] = see[i, k] = True
    P, s, V = spread(c, 0, see)
    P, s, V = P[:, 0], s[:, 0], V[0]
    O = P @ V
    two = torch.tensor(pairs, device="cuda")
    p, sv, v = P.gather(1, two), s.gather(1, two), V[two]                         # [n, 2], [n, 2], [n, 2, d]
    delta = (p[:, 0] * p[:, 1]) ** 2 * (sv ** 2).sum(-1) * ((v[:, 0] - v[:, 1]) ** 2).sum(-1)       # squared, for one unit of TERMS
    round2 = ONE ** 2 * ((p[..., None] * v) ** 2).sum() + ONE ** 2 * (O ** 2).sum()
    limit = (round2 + (2 * TERMS) ** 2 * delta.sum()).sqrt() + 2 * 7.5e-5 * O.norm()                 # (64 samples: twice the expected 2-norm)
    assert float(((7.8e-4 / 2) ** 2 * delta.sum()).sqrt()) > float(limit)         # half of what three terms would leave
    assert float((out - O).norm()) <= float(limit), (float((out - O).norm() / O.norm()), float(limit / O.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("n_q,n_kv,layout,n", [(32, 32, "freq1", 8), (32, 8, "freq1", 16), (32, 8, "freq2", 16), (16, 8, "band8", 3)])
@pytest.mark.parametrize("base", [100, 5000])
def test_equal_logits_give_the_exact_mean(n_q, n_kv, layout, n, base):
    """Tiles of several kv heads take every exponential from the hardware, which gives 1 for 0: with queries of zero all weights are 1, sums and
    result exact in 32 bits. Half of the values are 1, half 1 + 2^-7: the mean is a tie between two bf16 numbers and goes to the even one, 1;
    any weight off by 1e-5 would decide it."""
    c = Case(layer(n_q, n_kv, layout), [base], [n], mask="chain")
    c.q.zero_()
    s = c.slots(0, 0, base + n).long()
    c.cache.v[s // PAGE, :, s % PAGE, :] = (1.0 + (torch.arange(base + n, device="cuda") % 2) * 2.0 ** -7).to(torch.bfloat16)[:, None, None]
    out = c.run()
    even = [i for i in range(n) if (base + i + 1) % 2 == 0]                       # rows that see as many of one as of the other
    assert even and (out[even] == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n_q,n_kv,layout,v_bits", [(32, 8, "freq2", 0), (32, 32, "freq1", 0), (32, 8, "band8", 0), (32, 8, "freq2", 3)])
def test_one_token_a_sequence_is_decode_attention(n_q, n_kv, layout, v_bits):
    """A batch of which nobody drafts: the decode kernel's outputs (within 2e-3 of the formula in the 2-norm) to two roundings to bf16. The same in a
    workspace for the widest tree, which picks other tiles."""
    c = Case(layer(n_q, n_kv, layout), [1, 127, 128, 900, 3000, 2], [1] * 6, mask="chain", v_bits=v_bits)
    c.check(c.run())
    ws = c.pk.workspace(6, c.pk.default_splits(6, 3001))
    want = c.pk.decode(c.cache, c.q.float(), c.plan.positions, ws).double()
    wide = c.pk.tree_workspace(6, c.cap, 64, c.cache.max_pages * PAGE)
    for space in (c.ws, wide):
        out = c.pk.tree_step(c.cache, c.q, c.plan, space).double()
        assert float((out - want.view_as(out)).norm()) <= (2e-3 + NORM) * float(want.norm())
        assert int(space.status.abs().sum()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n_q,n_kv,layout,v_bits", [(32, 8, "freq2", 0), (32, 32, "freq1", 0), (32, 8, "freq2", 2)])
def test_small_trees_in_a_workspace_for_the_widest(n_q, n_kv, layout, v_bits):
    c = Case(layer(n_q, n_kv, layout), [700, 0, 255, 1500], [6, 1, 0, 17], v_bits=v_bits)
    c.ws = c.pk.tree_workspace(4, c.cap, 64, c.cache.max_pages * PAGE)
    c.check(c.run())
