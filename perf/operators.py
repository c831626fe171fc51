"""Speculative decoding on the paged latent cache: the operators of one step, with their plain forms.

A step of a server that drafts a tree of tokens for every sequence:

  plan   `PagedLatentCache.plan_step`: pages, slots, positions and ancestor masks of the step's tokens from the
         requests' lengths; `PagedLatentCache.truncate`: sequences cut to given lengths, their pages back to the pool
  tree   `PhasorKey.tree_step`: attention of every drafted token to its sequence's cached tokens and to the drafted
         tokens its mask names, on the NVFP4 latent pages
  keep   `PagedLatentCache.keep_rows`: the rows of the accepted path moved up behind the cached tokens, in every layer

`run` computes them with elementary torch operations in 32 bits, or (``own``) with this package's calls.
"""
import random

import torch

own = False

PAGE = 128                       # tokens per cache page
D = 128                          # head dimension
LOG2 = lambda r, lo, hi: int(round(2 ** r.uniform(lo, hi)))

# factor layouts of the package's own configurations: complex latent dims, real slow dims, slow frequencies
LAYOUTS = {"freq2": (128, 0, 0), "band8": (120, 16, 8), "freq1": (64, 0, 0)}


# ---------------------------------------------------------------------------------------------- cases
def _tree(name, layout, n_q, n_kv, batch, tokens, draft, v_bits=0, ragged=False, q="bf16", mask="tree"):
    return dict(name=name, op="tree", layout=layout, n_q=n_q, n_kv=n_kv, batch=batch, tokens=tokens, draft=draft,
                v_bits=v_bits, ragged=ragged, q=q, mask=mask)


def _plan(name, batch, cached, new, tree=False, ragged=True, pad=0):
    return dict(name=name, op="plan", batch=batch, cached=cached, new=new, tree=tree, ragged=ragged, pad=pad)


def _keep(name, layers, layout, n_kv, batch, tokens, draft, v_bits=0):
    return dict(name=name, op="keep", layers=layers, layout=layout, n_kv=n_kv, batch=batch, tokens=tokens, draft=draft, v_bits=v_bits)


def listed():
    return [
        # one user, a short prompt, a chain of five drafted tokens: latency is all there is
        _tree("tree_one_user", "freq2", 32, 8, 1, 300, 5, q="fp32", mask="chain"),
        # the benchmark's batch and context with 16 drafted tokens a sequence: the whole cache is read once
        _tree("tree_b16_t32768_n16", "freq2", 32, 8, 16, 32768, 16),
        # one long document, a small tree: the token axis has to be split over the GPU
        _tree("tree_t131072_n8", "freq2", 32, 8, 1, 131072, 8),
        # the widest tree a mask word holds: bound by arithmetic
        _tree("tree_b8_t8192_n64", "freq2", 32, 8, 8, 8192, 64),
        # band layout, a ragged batch as a server has it: odd lengths, some sequences without drafts
        _tree("tree_ragged_band8", "band8", 32, 8, 24, 7001, 21, ragged=True),
        # a query head per kv head (the 7B multi-head shape)
        _tree("tree_mha", "freq1", 32, 32, 4, 4096, 8),
        # value pages of three-bit codes
        _tree("tree_q3_b16_t16384", "freq2", 32, 8, 16, 16384, 12, v_bits=3),
        # decode bookkeeping of a batch: one token a sequence
        _plan("plan_decode", 64, 2000, 1, ragged=False),
        # a speculative step: trees of up to 32 tokens, a buffer padded for a captured graph
        _plan("plan_tree", 96, 9000, 32, tree=True, pad=64),
        # admission of 48 prompts
        _plan("plan_prefill", 48, 0, 8192),
        # the accepted path of one small batch in one layer
        _keep("keep_one_layer", 1, "freq2", 8, 4, 500, 8),
        # the accepted paths of a batch in eight layers that share the page table
        _keep("keep_eight_layers", 8, "freq2", 8, 48, 700, 32),
    ]


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "plan", "keep"])
    if kind == "plan":
        tree = rng.random() < 0.5
        new = LOG2(rng, 0, 6) if tree else LOG2(rng, 0, 13)
        return {k: v for k, v in _plan("", LOG2(rng, 0, 8) if tree or new < 256 else LOG2(rng, 0, 5.5), rng.choice([0, LOG2(rng, 0, 14)]), new, tree,
                                       rng.random() < 0.7, rng.choice([0, rng.randrange(1, 200)])).items() if k != "name"}
    layout = rng.choice(["freq2", "freq2", "band8", "freq1"])
    if kind == "keep":
        return {k: v for k, v in _keep("", rng.choice([1, 2, 4, 6]), layout, rng.choice([8, 4, 32]) if layout == "freq1" else rng.choice([8, 4]),
                                       LOG2(rng, 0, 5), LOG2(rng, 0, 10), LOG2(rng, 1, 6), rng.choice([0, 0, 3, 2])).items() if k != "name"}
    n_q, n_kv = rng.choice([(32, 32), (32, 8), (16, 16)]) if layout == "freq1" else rng.choice([(32, 8), (32, 4), (32, 8), (16, 8), (24, 8), (64, 8), (28, 4)])
    draft = LOG2(rng, 0, 6)
    batch = LOG2(rng, 0, 5)
    budget = 16 * 32768 * 16 * 32 // (n_q * draft * batch * (4 if n_kv == 32 else 1))          # never more than the largest listed case
    tokens = min(LOG2(rng, 0, 17), max(1, budget), 16 * 32768 // batch)
    return {k: v for k, v in _tree("", layout, n_q, n_kv, batch, tokens, draft, rng.choice([0, 0, 0, 3, 2]), rng.random() < 0.5,
                                   rng.choice(["bf16", "bf16", "fp32"]), rng.choice(["tree", "tree", "chain", "any"])).items() if k != "name"}


def _rng(case, salt):
    return random.Random("%s %s" % (sorted((k, v) for k, v in case.items() if k != "name"), salt))


def _lengths(case):
    """Cached tokens and drafted tokens of every sequence: a matter of the case, not of the seed."""
    r, B = _rng(case, "lengths"), case["batch"]
    if not case.get("ragged", True):
        return [case["tokens"]] * B, [case["draft"]] * B
    base = [case["tokens"]] + [r.randint(0, case["tokens"]) for _ in range(B - 1)]
    n = [case["draft"]] + [r.randint(0, case["draft"]) for _ in range(B - 1)]
    return base, n


def _new_tokens(case):
    r, B = _rng(case, "new"), case["batch"]
    return [case["new"]] * B if not case["ragged"] else [case["new"]] + [r.randint(0, case["new"]) for _ in range(B - 1)]


def _kept(case):
    """Accepted draft indices of every sequence, ascending (a path from the root)."""
    r, out = _rng(case, "kept"), []
    for n in _lengths(case)[1]:
        k = r.randint(0, n)
        out.append(sorted(r.sample(range(n), k)))
    return out


def _row_bytes(W, n_kv, v_bits):
    return W // 2 + W // 16 + n_kv * (66 if v_bits else 2 * D)


def _width(layout):
    R, R_s, _ = LAYOUTS[layout]
    return 2 * R + R_s


def work(case):
    if case["op"] == "plan":
        n, B = sum(_new_tokens(case)), case["batch"]
        pages = n / PAGE
        return {"bytes": 4.0 * (5 * B + 3 * n + 2 * pages) + (12.0 * n if case["tree"] else 0.0), "flops": 0.0}
    W = _width(case["layout"])
    if case["op"] == "keep":
        rows = sum(map(len, _kept(case)))
        return {"bytes": 2.0 * rows * _row_bytes(W, case["n_kv"], case["v_bits"]) * case["layers"] + 8.0 * case["batch"] + 4.0 * rows, "flops": 0.0}
    base, n = _lengths(case)
    cached = sum(b + m for b, m in zip(base, n) if m)
    N = sum(n)
    pairs = sum((b + m) * m for b, m in zip(base, n))
    return {"bytes": float(cached * _row_bytes(W, case["n_kv"], case["v_bits"]) + N * case["n_q"] * D * (2 + (2 if case["q"] == "bf16" else 4))),
            "flops": 2.0 * pairs * case["n_q"] * (W + D)}


# ---------------------------------------------------------------------------------------------- inputs
def _page_bytes(W):
    Wp = 128 if W <= 128 else 256
    return PAGE * Wp // 2 + Wp // 64 * 512


def _code_index(W, dev):
    """[128, row bytes]: where byte c of a row's codes lies in a page (the swizzle of a shared-memory operand)."""
    RB = 64 if W <= 128 else 128
    o = torch.arange(PAGE * RB, device=dev)
    return (o ^ ((o >> 3) & (0x70 if RB == 128 else 0x30))).view(PAGE, RB)


def _scale_index(W, dev):
    """[128, blocks]: where the scale byte of (row, 16-column block) lies in a page."""
    Wp = 128 if W <= 128 else 256
    r, j = torch.arange(PAGE, device=dev)[:, None], torch.arange(Wp // 16, device=dev)[None, :]
    return PAGE * Wp // 2 + (j // 4) * 512 + (r % 32) * 16 + (r // 32) * 4 + j % 4


def _vq_index(n_kv, dev):
    """[n_kv, 128, 64]: where byte c of the codes of (kv head, row) lies in a page of quantised values."""
    r, c = torch.arange(PAGE, device=dev)[:, None], torch.arange(64, device=dev)[None, :]
    o = r * 64 + (((c // 16) ^ ((r // 2) % 4)) * 16) + c % 16
    return torch.arange(n_kv, device=dev)[:, None, None] * 8192 + o


LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _codes(y):
    """E2M1 codes of y: the nearest level, the sign in bit 3."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=y.device)
    idx = torch.bucketize(y.abs(), mids).to(torch.uint8)
    return idx | ((y < 0) & (idx > 0)).to(torch.uint8) << 3


def _make_pools(g, n_pages, W, n_kv, v_bits, with_v=True):
    """Pages as a server's writes leave them: latent rows with a decaying spectrum, normal value rows."""
    dev = g.device
    Wp = 128 if W <= 128 else 256
    second = 0.02
    latent = torch.zeros((n_pages, _page_bytes(W)), dtype=torch.uint8, device=dev)
    sigma = torch.linspace(2.5, 0.5, Wp, device=dev)
    ci, si = _code_index(W, dev), _scale_index(W, dev)
    step = 512
    for p in range(0, n_pages, step):
        m = min(step, n_pages - p)
        rows = torch.randn((m, PAGE, Wp), generator=g, device=dev) * sigma
        rows[:, :, W:] = 0
        blk = rows.view(m, PAGE, Wp // 16, 16)
        scale = (blk.abs().amax(-1) / 6.0 / second).clamp(max=448.0).to(torch.float8_e4m3fn)
        q = _codes(blk / (scale.float() * second).clamp_min(1e-30)[..., None]).view(m, PAGE, Wp)
        latent[p:p + m, ci.reshape(-1)] = (q[..., 0::2] | q[..., 1::2] << 4).reshape(m, -1)
        latent[p:p + m, si.reshape(-1)] = scale.view(torch.uint8).reshape(m, -1)
    v = vq = None
    if with_v and v_bits:
        vq = torch.zeros((n_pages, n_kv * 8448), dtype=torch.uint8, device=dev)
        vi = _vq_index(n_kv, dev).reshape(-1)
        for p in range(0, n_pages, step):
            m = min(step, n_pages - p)
            x = torch.randn((m, n_kv, PAGE, D), generator=g, device=dev)
            s = (x.abs().amax(-1).clamp_min(1e-5) / (3.0 if v_bits == 3 else 1.5)).to(torch.bfloat16)
            y = x / s.float()[..., None]
            y = y.round().clamp(-4, 3) if v_bits == 3 else torch.where(y.abs() > 1, 1.5, 0.5) * torch.where(y < 0, -1.0, 1.0)
            c = _codes(y)
            vq[p:p + m, vi] = (c[..., 0::2] | c[..., 1::2] << 4).reshape(m, -1)
            vq[p:p + m, n_kv * 8192:] = s.view(torch.uint8).reshape(m, -1)
    elif with_v:
        v = torch.randn((n_pages, n_kv, PAGE, D), generator=g, device=dev).to(torch.bfloat16)
    return latent, v, vq, second


def _parents(r, n, mask):
    return [i - 1 if mask == "chain" else r.randint(max(-1, i - 6), i - 1) for i in range(n)]


def _mask_words(r, n, mask):
    """One 64-bit word a drafted token: its ancestors and itself, or (mask "any") whatever a caller may set, nothing among it."""
    if mask == "any":
        words = [r.choice([0, r.getrandbits(64), (1 << 64) - 1, 1 << i]) for i in range(n)]
    else:
        words = []
        for i, p in enumerate(_parents(r, n, mask)):
            words.append((words[p] if p >= 0 else 0) | 1 << i)
    return [w - (1 << 64) if w >= 1 << 63 else w for w in words]


def _depths(r, n, mask):
    d = []
    for p in _parents(r, n, mask):
        d.append(d[p] + 1 if p >= 0 else 0)
    return d


def _tables(g, B, max_pages, n_pages):
    perm = torch.randperm(n_pages, generator=g, device=g.device).to(torch.int32)
    return perm[:B * max_pages].view(B, max_pages).contiguous(), perm


def _cu(n, dev):
    out = [0]
    for m in n:
        out.append(out[-1] + m)
    return torch.tensor(out, dtype=torch.int32, device=dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    r = random.Random(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    B = case["batch"]
    st = {"case": case}
    if case["op"] == "plan":
        new = _new_tokens(case)
        base = [r.randint(case["cached"] // 2, case["cached"]) for _ in range(B)]
        max_pages = (case["cached"] + case["new"] + PAGE - 1) // PAGE + 1
        n_pages = B * max_pages + 3
        used = [(b + PAGE - 1) // PAGE for b in base]
        perm = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
        table = torch.full((B, max_pages), -1, dtype=torch.int32)
        at, perm_c = 0, perm.cpu()
        for b in range(B):
            table[b, :used[b]] = perm_c[at:at + used[b]]
            at += used[b]
        free = torch.full((n_pages + 1,), -1, dtype=torch.int32)
        free[0] = n_pages - at
        free[1:1 + n_pages - at] = perm_c[at:]
        cap = sum(new) + case["pad"]
        parents = [p for m in new for p in _parents(r, m, "tree")] + [-1] * case["pad"] if case["tree"] else None
        st.update(page_table=table.to(dev), seqlens=i32(base), free=free.to(dev), base=i32(base), n_new=i32(new), capacity=cap,
                  parents=None if parents is None else i32(parents), n_pages=n_pages,
                  cu=torch.zeros(B + 1, dtype=torch.int32, device=dev), seq=torch.zeros(cap, dtype=torch.int32, device=dev),
                  positions=torch.zeros(cap, dtype=torch.int32, device=dev), slots=torch.zeros(cap, dtype=torch.int32, device=dev),
                  mask=torch.zeros(cap, dtype=torch.int64, device=dev))
        if own:                                              # the cache whose tables these are, and the step's plan
            from phasorkv_b200 import PagedLatentCache
            cache = PagedLatentCache(128, 1, D, B, max_pages * PAGE, dev, with_v=False, n_pages=n_pages)
            cache.use_page_pool()
            cache.page_table.copy_(st["page_table"]), cache.seqlens.copy_(st["seqlens"]), cache.free.copy_(st["free"])
            st.update(cache=cache, plan=cache.step_plan(cap, tree=case["tree"]))
        return st

    W = _width(case["layout"])
    n_kv, v_bits = case["n_kv"], case["v_bits"]
    base, n = _lengths(case)
    max_pages = max((b + m + PAGE - 1) // PAGE for b, m in zip(base, n)) or 1
    n_pages = B * max_pages + 2
    table, _ = _tables(g, B, max_pages, n_pages)
    seqlens, cu = i32([b + m for b, m in zip(base, n)]), _cu(n, dev)
    N = sum(n)
    st.update(page_table=table, seqlens=seqlens, cu=cu, W=W, n_pages=n_pages, N=N)
    if case["op"] == "keep":
        kept = _kept(case)
        keep = torch.full((max(N, 1),), -1, dtype=torch.int32)
        for c, k in zip(cu.tolist(), kept):
            keep[c:c + len(k)] = i32(k).cpu()
        pools = [_make_pools(g, n_pages, W, n_kv, v_bits) for _ in range(case["layers"])]
        st.update(keep=keep.to(dev), n_keep=i32([len(k) for k in kept]), lengths=torch.zeros(B, dtype=torch.int32, device=dev),
                  latent=[p[0] for p in pools], v=[p[2] if v_bits else p[1] for p in pools])
        if own:                                              # the layers' caches; they share the first one's tables
            from phasorkv_b200 import PagedLatentCache
            caches = [PagedLatentCache(W, n_kv, D, B, max_pages * PAGE, dev, n_pages=n_pages, v_bits=v_bits) for _ in pools]
            for i, c in enumerate(caches):
                c.latent.copy_(st["latent"][i].view(-1))
                (c.vq if v_bits else c.v).view(-1).copy_(st["v"][i].view(-1))
                st["latent"][i], st["v"][i] = c.latent.view(n_pages, -1), (c.vq.view(n_pages, -1) if v_bits else c.v)
                if i:
                    c.share_pages(caches[0])
            caches[0].page_table.copy_(table), caches[0].seqlens.copy_(seqlens)
            plan = caches[0].step_plan(max(N, 1))
            plan.cu.copy_(cu)
            st.update(caches=caches, plan=plan)
        return st

    R, R_s, n_slow = LAYOUTS[case["layout"]]
    n_q, h2 = case["n_q"], D // 2
    latent, v, vq, second = _make_pools(g, n_pages, W, n_kv, v_bits)
    words, depth = [], []
    for m in n:
        s = r.getrandbits(32)
        words += _mask_words(random.Random(s), m, case["mask"])
        depth += _depths(random.Random(s), m, "chain" if case["mask"] == "any" else case["mask"])
    positions = [b + d for (b, m), ds in zip(zip(base, n), _split(depth, n)) for d in ds]
    A = torch.complex(torch.randn((n_kv, R), generator=g, device=dev), torch.randn((n_kv, R), generator=g, device=dev)) * 0.7071
    freq = (torch.arange(R, device=dev) * (h2 - n_slow)) // R
    st.update(latent=latent, v=v, vq=vq, second=second, A=A, freq=freq,
              A_s=torch.randn((n_kv, 2 * n_slow, R_s), generator=g, device=dev) * 0.25 if R_s else None,
              slow=torch.arange(h2 - n_slow, h2, device=dev),
              inv_freq=torch.pow(torch.tensor(500000.0, dtype=torch.float64, device=dev), -torch.arange(h2, dtype=torch.float64, device=dev) / h2),
              q=torch.randn((N, n_q, D), generator=g, device=dev).to(torch.bfloat16 if case["q"] == "bf16" else torch.float32),
              positions=i32(positions), mask=torch.tensor(words, dtype=torch.int64, device=dev), max_draft=max(n), max_tokens=max_pages * PAGE)
    if own:                                                  # the layer, its cache, the step's plan and the workspace
        from phasorkv_b200 import PagedLatentCache, PhasorKey
        pk = PhasorKey.from_factors(A.cpu(), torch.zeros((R, 16), dtype=torch.complex64), freq.cpu(), n_q, n_kv, D, st["inv_freq"].cpu(),
                                    None if not R_s else st["A_s"].cpu(), torch.zeros((R_s, 16)) if R_s else None, st["slow"].cpu())
        pk.set_second(second)
        cache = PagedLatentCache(W, n_kv, D, B, max_pages * PAGE, dev, n_pages=n_pages, v_bits=v_bits)
        cache.latent.copy_(latent.view(-1))
        if v_bits:
            cache.vq.copy_(vq.view(-1))
        else:
            cache.v.copy_(v)
        st["latent"] = st["v"] = st["vq"] = latent = v = vq = None
        cache.page_table.copy_(table), cache.seqlens.copy_(seqlens)
        plan = cache.step_plan(N, tree=True)
        plan.cu.copy_(cu), plan.positions.copy_(st["positions"]), plan.mask.copy_(st["mask"])
        st.update(pk=pk, cache=cache, plan=plan, ws=pk.tree_workspace(B, N, st["max_draft"], cache.max_pages * PAGE))
    return st


def _split(values, n):
    out, at = [], 0
    for m in n:
        out.append(values[at:at + m])
        at += m
    return out


# ---------------------------------------------------------------------------------------------- plain forms
def _latent_values(pages, W, second):
    """Latent pages [P, bytes] -> [P, 128, W] fp32."""
    dev = pages.device
    lut = torch.tensor(LEVELS + [-x for x in LEVELS], device=dev)
    c = pages[:, _code_index(W, dev).reshape(-1)].view(len(pages), PAGE, -1)
    val = lut[torch.stack([c & 15, c >> 4], dim=-1).long()].flatten(2)
    sc = pages[:, _scale_index(W, dev).reshape(-1)].view(torch.float8_e4m3fn).float().view(len(pages), PAGE, -1) * second
    return (val.view(len(pages), PAGE, -1, 16) * sc[..., None]).flatten(2)[:, :, :W]


def _vq_values(pages, n_kv):
    """Quantised value pages [P, bytes] -> [P, n_kv, 128, D] fp32."""
    dev = pages.device
    lut = torch.tensor(LEVELS + [-x for x in LEVELS], device=dev)
    c = pages[:, _vq_index(n_kv, dev).reshape(-1)].view(len(pages), n_kv, PAGE, 64)
    s = pages[:, n_kv * 8192:].contiguous().view(torch.bfloat16).view(len(pages), n_kv, PAGE).float()
    return lut[torch.stack([c & 15, c >> 4], dim=-1).long()].flatten(3) * s[..., None]


def _tree_plain(st):
    case, W, cu = st["case"], st["W"], st["cu"].long()
    dev = cu.device
    B, n_q, n_kv, N, n = case["batch"], case["n_q"], case["n_kv"], st["N"], st["max_draft"]
    R, h2, rep = st["A"].shape[1], D // 2, case["n_q"] // case["n_kv"]
    # the queries absorbed: [Re q' | Im q' | slow]
    ang = st["positions"].double()[:, None] * st["inv_freq"][None, :]
    ph = torch.polar(torch.ones_like(ang), ang).to(torch.complex64)
    q = st["q"].float()
    zq = torch.complex(q[..., :h2].contiguous(), q[..., h2:].contiguous()) * ph[:, None, :]
    kv = torch.arange(n_q, device=dev) // rep
    qp = st["A"].conj()[kv][None] * zq[:, :, st["freq"]]
    qa = torch.cat([qp.real, qp.imag], dim=-1)
    if st["A_s"] is not None:
        qs = torch.cat([q[..., st["slow"]], q[..., st["slow"] + h2]], dim=-1)
        qa = torch.cat([qa, torch.einsum("nhs,hsr->nhr", qs, st["A_s"][kv])], dim=-1)
    # every sequence's queries and pages, padded to the longest
    i = torch.arange(N, device=dev)
    seq = torch.searchsorted(cu[1:], i, right=True)
    row = i - cu[seq]
    Q = torch.zeros((B, n, n_q, W), device=dev)
    Q[seq, row] = qa
    words = torch.zeros((B, n), dtype=torch.int64, device=dev)
    words[seq, row] = st["mask"]
    pt = st["page_table"].long()
    C = _latent_values(st["latent"], W, st["second"])[pt].flatten(1, 2)
    S = torch.einsum("bnhw,btw->bhnt", Q, C) * D ** -0.5
    # what a drafted token sees: all cached tokens, and the drafted ones its word names
    T = C.shape[1]
    t = torch.arange(T, device=dev)
    m = cu[1:] - cu[:-1]
    base = st["seqlens"].long() - m
    j = t[None, :] - base[:, None]
    bit = (words[:, :, None] >> j.clamp(0, 63)[:, None, :]) & 1
    see = (j < 0)[:, None, :] | (((j >= 0) & (j < m[:, None]))[:, None, :] & (bit == 1))
    S = S.masked_fill_(~see[:, None], float("-inf"))
    top = S.amax(-1, keepdim=True)
    P = torch.exp(S - torch.where(torch.isinf(top), 0.0, top))
    del S
    den = P.sum(-1, keepdim=True)
    V = (_vq_values(st["vq"], n_kv) if case["v_bits"] else st["v"].float())[pt].transpose(1, 2).flatten(2, 3)      # [B, n_kv, T, D]
    O = P.view(B, n_kv, rep * n, T) @ V
    O = O.view(B, n_q, n, D) / torch.where(den > 0, den, 1.0)
    return {"out": O.transpose(1, 2)[seq, row].to(torch.bfloat16)}


def _plan_plain(st):
    case = st["case"]
    dev = st["cu"].device
    cap = st["capacity"]
    base, new, table, free = st["seqlens"].long(), st["n_new"].long(), st["page_table"], st["free"]
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), new.cumsum(0)])
    total = base + new
    had, want = (base + PAGE - 1) // PAGE, (total + PAGE - 1) // PAGE
    off = (want - had).cumsum(0) - (want - had)
    p = torch.arange(table.shape[1], device=dev)
    fresh = (p >= had[:, None]) & (p < want[:, None])
    k = off[:, None] + p - had[:, None]
    st["page_table"] = table = torch.where(fresh, free[(free[0] - k).clamp(0, len(free) - 1)], table)
    count = free[0] - (want - had).sum()
    st["free"] = free = torch.where(torch.arange(len(free), device=dev) == 0, count, free).to(torch.int32)
    i = torch.arange(cap, device=dev)
    live = i < cu[-1]
    seq = torch.searchsorted(cu[1:], i, right=True).clamp(max=len(new) - 1)
    at = i - cu[seq]
    local = base[seq] + at
    slots = table[seq, (local // PAGE).clamp(max=table.shape[1] - 1)] * PAGE + local % PAGE
    mask = None
    if case["tree"]:
        # ancestors: the parent relation closed by doubling (a path has at most 64 tokens)
        n = 64
        par = torch.full((len(new), n + 1), n, dtype=torch.long, device=dev)          # row n: the root's parent is itself
        up = torch.where(st["parents"][:cap].long() < 0, n, st["parents"][:cap].long())
        par[seq[live], at[live]] = up[live]
        word = (1 << torch.arange(n, device=dev)).expand(len(new), n)
        word = torch.cat([word, torch.zeros((len(new), 1), dtype=torch.long, device=dev)], 1)
        depth = torch.cat([torch.ones((len(new), n), dtype=torch.long, device=dev), torch.zeros((len(new), 1), dtype=torch.long, device=dev)], 1)
        for _ in range(6):
            word, depth, par = word | word.gather(1, par), depth + depth.gather(1, par), par.gather(1, par)
        row = at.clamp(0, n - 1)
        mask = torch.where(live, word[seq, row], st["mask"])
        local = base[seq] + depth[seq, row] - 1
    out = {"cu": cu.to(torch.int32), "seq": torch.where(live, seq, st["seq"]).to(torch.int32),
           "positions": torch.where(live, local, st["positions"]).to(torch.int32), "slots": torch.where(live, slots, -1).to(torch.int32)}
    if mask is not None:
        out["mask"] = mask
    # the step is dropped again: back to the lengths before it
    have = total
    left = torch.minimum(have, st["base"].long())
    had, want = (left + PAGE - 1) // PAGE, (have + PAGE - 1) // PAGE
    off = (want - had).cumsum(0) - (want - had)
    gone = (p >= had[:, None]) & (p < want[:, None])
    K = (want - had).sum()
    at = torch.where(gone, free[0] + K - (off[:, None] + p - had[:, None]), len(free))
    free = torch.cat([free, free.new_zeros(1)]).scatter(0, at.reshape(-1), table.reshape(-1))[:-1]
    st["free"] = torch.where(torch.arange(len(free), device=dev) == 0, free[0] + K, free).to(torch.int32)
    st["page_table"] = torch.where(gone, -1, table)
    st["seqlens"] = left.to(torch.int32)
    return dict(out, page_table=st["page_table"], free=st["free"], seqlens=st["seqlens"])


def _keep_plain(st):
    case, W = st["case"], st["W"]
    dev, B = st["cu"].device, case["batch"]
    cu = st["cu"].long()
    base = st["seqlens"].long() - (cu[1:] - cu[:-1])
    nk = st["n_keep"].long()
    total = torch.repeat_interleave(torch.arange(B, device=dev), nk)
    j = torch.arange(len(total), device=dev) - (nk.cumsum(0) - nk)[total]
    src = base[total] + st["keep"].long()[cu[total] + j]
    dst = base[total] + j
    pt = st["page_table"].long()
    sp, sr, dp, dr = pt[total, src // PAGE], src % PAGE, pt[total, dst // PAGE], dst % PAGE
    bytes_of = torch.cat([_code_index(W, dev), _scale_index(W, dev)], dim=1)
    if case["v_bits"]:
        n_kv = case["n_kv"]
        s = n_kv * 8192 + torch.arange(n_kv, device=dev)[:, None, None] * 256 + torch.arange(PAGE, device=dev)[None, :, None] * 2 + torch.arange(2, device=dev)
        v_of = torch.cat([_vq_index(n_kv, dev), s], dim=2).transpose(0, 1).flatten(1)
    for i in range(case["layers"]):
        pool = st["latent"][i]
        pool[dp[:, None], bytes_of[dr]] = pool[sp[:, None], bytes_of[sr]]
        v = st["v"][i]
        if case["v_bits"]:
            v[dp[:, None], v_of[dr]] = v[sp[:, None], v_of[sr]]
        else:
            v[dp, :, dr] = v[sp, :, sr]
    return {"lengths": (base + nk).to(torch.int32), "latent": st["latent"], "v": st["v"]}


# ---------------------------------------------------------------------------------------------- one pass
def run(st):
    """One pass. A plan is dropped again at its end, so that the next pass finds the lengths it starts from; the rows
    that `keep` moves are bytes, and come back as the pools that hold them."""
    op = st["case"]["op"]
    if not own:
        return {"tree": _tree_plain, "plan": _plan_plain, "keep": _keep_plain}[op](st)
    if op == "tree":
        out = torch.empty(st["q"].shape, dtype=torch.bfloat16, device=st["q"].device)
        st["pk"].tree_step(st["cache"], st["q"], st["plan"], st["ws"], out)
        return {"out": out}
    if op == "keep":
        st["caches"][0].keep_rows(st["plan"], st["keep"], st["n_keep"], st["lengths"], layers=st["caches"])
        return {"lengths": st["lengths"], "latent": st["latent"], "v": st["v"]}
    cache, plan = st["cache"], st["plan"]
    cache.plan_step(plan, st["n_new"], parents=st["parents"])
    cache.truncate(st["base"])
    out = {"cu": plan.cu, "seq": plan.seq, "positions": plan.positions, "slots": plan.slots}
    if st["case"]["tree"]:
        out["mask"] = plan.mask
    return dict(out, page_table=cache.page_table, free=cache.free, seqlens=cache.seqlens)


# ---------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The definitions once more, sequence by sequence, in doubles and Python integers."""
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "tree":
        return _tree_exact(st)
    if case["op"] == "keep":
        return _keep_exact(st)
    return _plan_exact(st)


def _tree_exact(st):
    case, W, cu = st["case"], st["W"], st["cu"].tolist()
    n_q, n_kv = case["n_q"], case["n_kv"]
    dev = st["q"].device
    out = torch.zeros((st["N"], n_q, D), dtype=torch.float64, device=dev)
    mag = lambda c: torch.where(c < 2, c * 0.5, torch.pow(2.0, (c >> 1).double() - 1) * (1 + 0.5 * (c & 1)))
    number = lambda c: torch.where(c > 7, -1.0, 1.0) * mag(c & 7)
    ci, si = _code_index(W, dev), _scale_index(W, dev)
    for b in range(case["batch"]):
        m, T = cu[b + 1] - cu[b], int(st["seqlens"][b])
        if m == 0:
            continue
        pages = st["page_table"][b, :(T + PAGE - 1) // PAGE].long()
        raw = st["latent"][pages].int()
        c = raw[:, ci]
        c = torch.stack([c % 16, c // 16], dim=-1).flatten(2)
        e = raw[:, si]
        scale = torch.where(e < 8, e * 2.0 ** -9, torch.pow(2.0, (e >> 3).double() - 7) * (1 + (e & 7) / 8.0))
        rows = (number(c).unflatten(2, (-1, 16)) * (scale * st["second"])[..., None]).flatten(2).flatten(0, 1)[:T, :W]
        if case["v_bits"]:
            raw = st["vq"][pages]
            c = raw[:, _vq_index(n_kv, dev)].int()
            s = raw[:, n_kv * 8192:].contiguous().view(torch.bfloat16).double().view(len(pages), n_kv, PAGE, 1)
            V = (number(torch.stack([c % 16, c // 16], dim=-1).flatten(3)) * s).transpose(0, 1).flatten(1, 2)[:, :T]
        else:
            V = st["v"][pages].double().transpose(0, 1).flatten(1, 2)[:, :T]
        words = [w % (1 << 64) for w in st["mask"][cu[b]:cu[b + 1]].tolist()]
        base = T - m
        see = torch.ones((m, T), dtype=torch.bool)
        for x in range(m):
            see[x, base:] = torch.tensor([bool(words[x] >> y & 1) for y in range(m)])
        see = see.to(dev)
        q = st["q"][cu[b]:cu[b + 1]].double()
        ang = st["positions"][cu[b]:cu[b + 1]].double()[:, None] * st["inv_freq"]
        cs, sn = ang.cos()[:, None], ang.sin()[:, None]
        re, im = q[..., :D // 2], q[..., D // 2:]
        zr, zi = (re * cs - im * sn)[..., st["freq"]], (re * sn + im * cs)[..., st["freq"]]
        for g in range(n_kv):
            hs = slice(g * (n_q // n_kv), (g + 1) * (n_q // n_kv))
            ar, ai = st["A"][g].real.double(), st["A"][g].imag.double()
            qa = [ar * zr[:, hs] + ai * zi[:, hs], ar * zi[:, hs] - ai * zr[:, hs]]
            if st["A_s"] is not None:
                qa.append(torch.cat([re[:, hs][..., st["slow"]], im[:, hs][..., st["slow"]]], dim=-1) @ st["A_s"][g].double())
            s = torch.cat(qa, dim=-1) @ rows.T / D ** 0.5
            s = s.masked_fill(~see[:, None], -torch.inf)
            p = torch.softmax(s, dim=-1).nan_to_num(0.0) if (~see.any(1)).any() else torch.softmax(s, dim=-1)
            out[cu[b]:cu[b + 1], hs] = p @ V[g]
    return {"out": out}


def _plan_exact(st):
    case = st["case"]
    base, new, free = st["seqlens"].tolist(), st["n_new"].tolist(), st["free"].tolist()
    table = st["page_table"].tolist()
    cap = st["capacity"]
    cu, seq, pos, slots, mask = [0], [0] * cap, [0] * cap, [-1] * cap, [0] * cap
    stack, taken, at = free[1:1 + free[0]], [], 0
    parents = st["parents"].tolist() if st["parents"] is not None else None
    for b, (L, m) in enumerate(zip(base, new)):
        for p in range((L + PAGE - 1) // PAGE, (L + m + PAGE - 1) // PAGE):
            table[b][p] = stack.pop()
            taken.append((b, p))
        depth = []
        for i in range(m):
            t = L + i
            seq[at], pos[at], slots[at] = b, t, table[b][t // PAGE] * PAGE + t % PAGE
            if parents is not None:
                up = parents[at]
                depth.append(0 if up < 0 else depth[up] + 1)
                mask[at] = (mask[at - i + up] if up >= 0 else 0) | 1 << i
                pos[at] = L + depth[i]
            at += 1
        cu.append(at)
    for b, p in reversed(taken):
        stack.append(table[b][p])
        table[b][p] = -1
    mask = [w - (1 << 64) if w >= 1 << 63 else w for w in mask]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    out = {"cu": i32(cu), "seq": i32(seq), "positions": i32(pos), "slots": i32(slots)}
    if parents is not None:
        out["mask"] = torch.tensor(mask, dtype=torch.int64)
    return dict(out, page_table=i32(table), free=i32([len(stack)] + stack + free[1 + len(stack):]), seqlens=i32(base))


def _keep_exact(st):
    case, W, cu = st["case"], st["W"], st["cu"].tolist()
    n_kv = case["n_kv"]
    lens, keep, nk, table = st["seqlens"].tolist(), st["keep"].tolist(), st["n_keep"].tolist(), st["page_table"].tolist()
    RB, blocks = (64, 8) if W <= 128 else (128, 16)
    moves = []
    for b in range(case["batch"]):
        base = lens[b] - (cu[b + 1] - cu[b])
        for j in range(nk[b]):
            moves.append([(table[b][t // PAGE], t % PAGE) for t in (base + keep[cu[b] + j], base + j)])
    code = lambda r: [r * RB + ((c // 16) ^ (r % 8 if RB == 128 else r // 2 % 4)) * 16 + c % 16 for c in range(RB)]
    scale = lambda r: [PAGE * RB + j // 4 * 512 + r % 32 * 16 + r // 32 * 4 + j % 4 for j in range(blocks)]
    place = {r: torch.tensor(code(r) + scale(r)) for r in range(PAGE)}
    if case["v_bits"]:
        vplace = {r: torch.tensor([g * 8192 + r * 64 + ((c // 16) ^ (r // 2 % 4)) * 16 + c % 16 for g in range(n_kv) for c in range(64)] +
                                  [n_kv * 8192 + g * 256 + 2 * r + k for g in range(n_kv) for k in (0, 1)]) for r in range(PAGE)}
    latent, v = [x.cpu() for x in st["latent"]], [x.cpu() for x in st["v"]]
    for i in range(case["layers"]):
        for (sp, sr), (dp, dr) in moves:
            latent[i][dp, place[dr]] = latent[i][sp, place[sr]]
            if case["v_bits"]:
                v[i][dp, vplace[dr]] = v[i][sp, vplace[sr]]
            else:
                v[i][dp, :, dr] = v[i][sp, :, sr]
    return {"lengths": torch.tensor([lens[b] - cu[b + 1] + cu[b] + nk[b] for b in range(case["batch"])], dtype=torch.int32),
            "latent": latent, "v": [x if case["v_bits"] else x.double() for x in v]}
