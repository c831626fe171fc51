"""CPU oracle for the PhasorKey decode path. TEST INFRASTRUCTURE ONLY.

This file restates, in plain torch-CPU arithmetic, what the reference computes on the path this
repository accelerates. Only the test suite, the smoke check and the CPU-baseline leg of the
benchmark may import it; the product (the CUDA library and its Python host) never does.

Pinned: every function here is checked against vectors produced by the reference itself
(tests/golden/*.npz, generated by tests/golden/make_golden.py from an unmodified import of the
reference), including the reference's one published identity for this path ("PhasorKey scores
equal keys rebuilt from W_hat and rotated by HF's apply_rotary_pos_emb", README.md:75-77).

Reference anchors (file:line are paths inside the reference project):
  rope_phasors      phasorkv/rope.py:23-32
  to_complex        phasorkv/rope.py:12-15
  PhasorKeyOracle   phasorkv/latent.py:27-88   (write :61-70, absorb :72-83, scores :85-88)
  nvfp4_*           phasorkv/quant.py:70-124, phasorkv/kernels/nvfp4.py:17-55
  quantize_per_token  phasorkv/kernels/nvfp4.py:58-67 (per-token low-bit V tiers)
  attend            phasorkv/metrics.py:23,29-35 ; phasorkv/kernels/latent_attn.py:682-685
  merge_partials    phasorkv/kernels/dense_attn.py:72-74
  w_hat / hf_rope   phasorkv/factorize.py:149-163 ; phasorkv/rope.py:35-38 ; engine.py:108-112
"""
from __future__ import annotations

import math

import torch

E2M1_LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E2M1_MIDS = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
E4M3_MAX = 448.0
E2M1_MAX = 6.0
LOG2E = 1.4426950408889634


# ----------------------------------------------------------------------------------------------
# phasors and layout (phasorkv/rope.py)
# ----------------------------------------------------------------------------------------------

def rope_phasors(inv_freq: torch.Tensor, positions: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """scale * e^{i * t * inv_freq[j]} as complex128 [len(positions), h]; the angle is formed in
    float64 exactly as rope.py:29-32 does."""
    ang = positions.to(torch.float64)[:, None] * inv_freq.to(torch.float64)[None, :]
    return torch.polar(torch.full_like(ang, float(scale)), ang)


def to_complex(x: torch.Tensor) -> torch.Tensor:
    """rotate-half layout [..., d] -> complex [..., d/2]: z_j = x[j] + i x[j + d/2] (rope.py:12-15)."""
    h = x.shape[-1] // 2
    return torch.complex(x[..., :h].contiguous(), x[..., h:].contiguous())


# ----------------------------------------------------------------------------------------------
# PhasorKey (phasorkv/latent.py)
# ----------------------------------------------------------------------------------------------

def _product(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """a @ b. Small fp32 products add up over the inner index, one fused multiply-add after the other, as the stored vectors were formed: host
    libraries differ in their order, by a last bit. (A product of fp32 numbers is exact in fp64.) Larger ones, which are only
    held to tolerances, are the host library's."""
    if a.dtype != torch.float32 or b.dtype != torch.float32 or a.numel() * b.shape[-1] > 1 << 22:
        return a @ b
    c = torch.zeros((*a.shape[:-1], b.shape[-1]), dtype=torch.float32)
    a, b = a.double(), b.double()
    for k in range(a.shape[-1]):
        c = (a[..., k:k + 1] * b[k] + c.double()).float()
    return c


class PhasorKeyOracle:
    """write / absorb / scores on injected factors (the attributes latent.py:47-54 builds)."""

    def __init__(self, A, B, freq, n_q, n_kv, head_dim, A_s=None, B_s=None, slow=None):
        self.A, self.B, self.freq = A, B, freq.long()
        self.A_s, self.B_s = A_s, B_s
        self.slow = slow.long() if slow is not None else torch.zeros(0, dtype=torch.long)
        self.n_q, self.n_kv, self.h = n_q, n_kv, head_dim // 2
        self.R = B.shape[0]
        self.R_s = 0 if B_s is None else B_s.shape[0]

    @classmethod
    def from_spec(cls, spec, dtype=None):
        A, B = spec.A, spec.B
        A_s, B_s = spec.A_s, spec.B_s
        if dtype == torch.float64:
            A, B = A.to(torch.complex128), B.to(torch.complex128)
            A_s = None if A_s is None else A_s.double()
            B_s = None if B_s is None else B_s.double()
        return cls(A, B, spec.freq, spec.n_q, spec.n_kv, spec.head_dim, A_s, B_s, spec.slow)

    @property
    def cache_width(self) -> int:
        return 2 * self.R + self.R_s

    def write(self, x: torch.Tensor, ph: torch.Tensor) -> torch.Tensor:
        """x [T, D], ph [T, h] -> rows [T, 2R + R_s] laid out [Re c_rot | Im c_rot | slow]."""
        rd = torch.float64 if x.dtype == torch.float64 else torch.float32
        xr = x.to(rd)
        re = _product(xr, self.B.real.to(rd).T)
        im = _product(xr, self.B.imag.to(rd).T)
        c = torch.complex(re, im) * ph[:, self.freq].to(torch.complex128 if rd == torch.float64 else torch.complex64)
        out = [c.real, c.imag]
        if self.R_s:
            out.append(_product(xr, self.B_s.to(rd).T))
        return torch.cat(out, dim=-1)

    def absorb(self, q: torch.Tensor, ph: torch.Tensor) -> torch.Tensor:
        """q [H, Tq, d] pre-RoPE, ph [Tq, h] -> [H, Tq, 2R + R_s]."""
        zq = to_complex(q)
        zq = zq * ph.to(zq.dtype)
        g = torch.arange(self.n_q) // (self.n_q // self.n_kv)
        Ah = self.A[g].conj().to(zq.dtype)
        qp = Ah[:, None, :] * zq[:, :, self.freq]
        out = [qp.real, qp.imag]
        if self.R_s:
            qs = torch.cat([q[..., self.slow], q[..., self.slow + self.h]], dim=-1)
            out.append(torch.einsum("htr,hrk->htk", qs, self.A_s[g].to(q.dtype)))
        return torch.cat(out, dim=-1)

    @staticmethod
    def scores(q_abs: torch.Tensor, cache: torch.Tensor) -> torch.Tensor:
        """Unscaled logits [H, Tq, Tk]."""
        return _product(q_abs, cache.T.to(q_abs.dtype))


# ----------------------------------------------------------------------------------------------
# NVFP4 (phasorkv/quant.py, phasorkv/kernels/nvfp4.py)
# ----------------------------------------------------------------------------------------------

def cast_e4m3(x: torch.Tensor, up: bool = False) -> torch.Tensor:
    """Non-negative scales to E4M3 by round-to-nearest-even after clamping to [0, 448] (quant.py:84).
    up=True (PHASORKV_SCALE_UP=1 in the reference, quant.py:57,85-88): a scale that was rounded down is
    moved one E4M3 step up, so the block's largest element is never clipped."""
    y8 = x.clamp(0, E4M3_MAX).to(torch.float8_e4m3fn)
    if not up:
        return y8
    y = y8.float()
    e = torch.floor(torch.log2(y.clamp_min(2.0 ** -9)))
    ulp = torch.exp2(torch.clamp(e, min=-6) - 3)                       # subnormals: 2^-9
    return torch.where(y < x, (y + ulp).clamp(max=E4M3_MAX), y).to(torch.float8_e4m3fn)


def round_e2m1(y: torch.Tensor):
    """|y| to the E2M1 grid, saturating; exact midpoints go to the LOWER magnitude because the
    reference counts midpoints strictly below |y| (quant.py:75-78). -> (magnitude index, value)."""
    idx = torch.bucketize(y.abs().contiguous(), E2M1_MIDS.to(y.dtype))
    return idx, torch.sign(y) * E2M1_LEVELS.to(y.dtype)[idx]


def nvfp4_quantize(x: torch.Tensor, second: torch.Tensor, scale_up: bool = False):
    """Block-16 NVFP4 of x[..., n] along the last axis (nvfp4.py:43-55).

    -> codes uint8 [..., n] (bit 3 sign, bits 0-2 magnitude index; a value that rounds to zero
       never carries a sign), scale bytes uint8 [..., n/16] (E4M3 bit patterns), x_hat fp32."""
    assert x.shape[-1] % 16 == 0
    # one tensor scale, or one per 16-column block: the reference quantises tier by tier, each span of the row
    # with its own static scale (phasorkv/kernels/latent_attn.py:255-262)
    second = torch.as_tensor(second, dtype=torch.float32).reshape(-1)
    second = second.reshape(1) if second.numel() == 1 else second.reshape(-1, 1)
    xb = x.float().reshape(*x.shape[:-1], -1, 16)
    amax = xb.abs().amax(-1, keepdim=True)
    s8 = cast_e4m3(amax / E2M1_MAX / second, up=scale_up)
    scale = s8.float() * second
    idx, v = round_e2m1(xb / scale.clamp_min(1e-30))
    live = scale > 0
    idx = torch.where(live, idx, torch.zeros_like(idx))
    v = torch.where(live, v, torch.zeros_like(v))
    codes = (idx | ((v < 0).to(idx.dtype) << 3)).to(torch.uint8).reshape(x.shape)
    return codes, s8.squeeze(-1).view(torch.uint8), (v * scale).reshape(x.shape)


def pack_nibbles(codes: torch.Tensor) -> torch.Tensor:
    """Two codes per byte, even column in the low nibble (nvfp4.py:34-36)."""
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def unpack_nibbles(packed: torch.Tensor) -> torch.Tensor:
    return torch.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], -1)


def nvfp4_dequantize(codes: torch.Tensor, scale_bytes: torch.Tensor, second) -> torch.Tensor:
    """value(code) * (e4m3 scale * second), the x_hat of nvfp4.py:55."""
    second = torch.as_tensor(second, dtype=torch.float32).reshape(-1)
    second = second.reshape(1) if second.numel() == 1 else second.reshape(-1, 1)
    lv = torch.cat([E2M1_LEVELS, -E2M1_LEVELS])
    v = lv[codes.long()].reshape(*codes.shape[:-1], -1, 16)
    scale = scale_bytes.view(torch.float8_e4m3fn).float()[..., None] * second
    return (v * scale).reshape(codes.shape)


def nv_static_second(var: torch.Tensor) -> torch.Tensor:
    """Static tensor scale: 32 sigma of the widest channel over (448 * 6) (quant.py:119-124)."""
    top = var.max().clamp_min(1e-30)
    # (through fp64, which rounds an fp32 root correctly: some host libraries' fp32 roots are off by a bit)
    return (32 * top.double().sqrt().to(top.dtype) / (E4M3_MAX * E2M1_MAX)).reshape(1).float()


# ----------------------------------------------------------------------------------------------
# per-token low-bit V tiers (phasorkv/kernels/nvfp4.py:58-67)
# ----------------------------------------------------------------------------------------------

def e2m1_encode(v: torch.Tensor) -> torch.Tensor:
    """Exact E2M1 values -> 4-bit codes, sign in bit 3 (nvfp4.py:21-27; here -0.0 never occurs)."""
    idx = torch.bucketize(v.abs().contiguous(), E2M1_MIDS.to(v.dtype))
    assert torch.equal(E2M1_LEVELS.to(v.dtype)[idx], v.abs()), "value is not an exact E2M1 level"
    return (idx | ((v < 0).to(idx.dtype) << 3)).to(torch.uint8)


def e2m1_decode(codes: torch.Tensor) -> torch.Tensor:
    return torch.cat([E2M1_LEVELS, -E2M1_LEVELS])[codes.long()]


def quantize_per_token(x: torch.Tensor, nbits: int):
    """One bf16 scale per row of x[..., n] (nvfp4.py:58-67): 3 bits -> integers -4 .. 3 with
    scale = bf16(max(amax, 1e-5) / 3), round half to even; 2 bits -> levels +-0.5, +-1.5 with
    scale = bf16(max(amax, 1e-5) / 1.5), |y| <= 1 to 0.5 (quant.py:70-78 on the int2 grid).
    -> (E2M1 codes uint8 [..., n], bf16 scale [...], x_hat fp32 = value * scale)."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True).clamp_min(1e-5)
    if nbits == 2:
        s = (amax / 1.5).to(torch.bfloat16).float()
        y = x / s
        a = torch.where(y.abs() > 1.0, torch.full_like(y, 1.5), torch.full_like(y, 0.5))
        v = torch.where(y < 0, -a, a)
    else:
        qmax = 2 ** (nbits - 1) - 1
        s = (amax / qmax).to(torch.bfloat16).float()
        v = torch.round(x / s).clamp(-(2 ** (nbits - 1)), qmax)
    return e2m1_encode(v), s.squeeze(-1).to(torch.bfloat16), v * s


# ----------------------------------------------------------------------------------------------
# softmax . V and the split merge
# ----------------------------------------------------------------------------------------------

def attend(S: torch.Tensor, V: torch.Tensor, n_kv: int, head_dim: int) -> torch.Tensor:
    """S [H, Tk] unscaled logits of one decode query, V [Tk, n_kv, d] -> O [H, d] fp32.
    P = softmax(S * d^-0.5); V expanded over heads by repeat_interleave (metrics.py:23,29-35)."""
    H = S.shape[0]
    P = torch.softmax(S.float() * head_dim ** -0.5, dim=-1)
    Vh = V.float().transpose(0, 1).repeat_interleave(H // n_kv, dim=0)       # [H, Tk, d]
    return torch.einsum("ht,htd->hd", P, Vh)


def partial_attend(S: torch.Tensor, V: torch.Tensor, n_kv: int, head_dim: int):
    """One split's (m, l, o) in base 2: m = max log2-domain logit, l = sum 2^(s-m), o = sum 2^(s-m) v."""
    H = S.shape[0]
    s2 = S.float() * (LOG2E * head_dim ** -0.5)
    m = s2.amax(-1)
    p = torch.exp2(s2 - m[:, None])
    Vh = V.float().transpose(0, 1).repeat_interleave(H // n_kv, dim=0)
    return m, p.sum(-1), torch.einsum("ht,htd->hd", p, Vh)


def merge_partials(m: torch.Tensor, l: torch.Tensor, o: torch.Tensor) -> torch.Tensor:
    """m, l [S, H], o [S, H, d] -> O [H, d]: w_s = 2^(m_s - max m); O = sum w o / sum w l
    (dense_attn.py:72-74)."""
    M = m.amax(0, keepdim=True)
    w = torch.exp2(m - M)
    return (w[..., None] * o).sum(0) / (w * l).sum(0)[..., None]


# ----------------------------------------------------------------------------------------------
# the "rebuild keys with W_hat, then HF rotary" cross-check
# ----------------------------------------------------------------------------------------------

def w_hat(A, B, freq, n_kv, head_dim, A_s=None, B_s=None, slow=None) -> torch.Tensor:
    """Dense real key projection [n_kv*d, D] (float64) equivalent to the factors: per frequency j,
    M_hat_j = A_j B_j, real part to row g*d + j and imaginary part to row g*d + j + d/2
    (factorize.py:149-163); the slow block fills rows (g*d + s, g*d + s + d/2) for s in slow."""
    d, h = head_dim, head_dim // 2
    A = A.to(torch.complex128)
    B = B.to(torch.complex128)
    W = torch.zeros(n_kv * d, B.shape[1], dtype=torch.float64)
    heads = torch.arange(n_kv) * d
    for j in range(h):
        sel = (freq == j).nonzero().flatten()
        if sel.numel() == 0:
            continue
        M = A[:, sel] @ B[sel]
        W[heads + j] = M.real
        W[heads + j + h] = M.imag
    if B_s is not None:
        rows = torch.cat([heads[:, None] + slow[None, :], heads[:, None] + slow[None, :] + h], dim=1)  # [n_kv, 2 n_slow]
        M = A_s.double() @ B_s.double()                                         # [n_kv, 2 n_slow, D]
        W[rows.reshape(-1)] = M.reshape(-1, B.shape[1])
    return W


def hf_rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """HF Llama rotary on the last axis: x*cos + rotate_half(x)*sin, rotate_half(x) = [-x2, x1]."""
    h = x.shape[-1] // 2
    rot = torch.cat([-x[..., h:], x[..., :h]], dim=-1)
    return x * cos + rot * sin


def rebuilt_scores(W, x, q, ph_k, ph_q, n_q, n_kv, head_dim, slow=None) -> torch.Tensor:
    """Scores [H, Tq, Tk] from dense keys k = x W^T rotated with HF's rotary; frequencies in `slow`
    are left unrotated on both sides with the same magnitude (engine.py:108-112)."""
    T = x.shape[0]
    if slow is not None and slow.numel():
        ph_k, ph_q = ph_k.clone(), ph_q.clone()
        mag = ph_k[0, 0].abs()
        ph_k[:, slow] = mag.to(ph_k.dtype)
        ph_q[:, slow] = mag.to(ph_q.dtype)
    k = (x.double() @ W.T).reshape(T, n_kv, head_dim).transpose(0, 1)          # [n_kv, T, d]
    cos_k, sin_k = torch.cat([ph_k.real, ph_k.real], -1), torch.cat([ph_k.imag, ph_k.imag], -1)
    cos_q, sin_q = torch.cat([ph_q.real, ph_q.real], -1), torch.cat([ph_q.imag, ph_q.imag], -1)
    kr = hf_rotate(k, cos_k[None], sin_k[None])
    qr = hf_rotate(q.double(), cos_q[None], sin_q[None])                        # [H, Tq, d]
    kr = kr.repeat_interleave(n_q // n_kv, dim=0)
    return qr @ kr.transpose(1, 2)


# ----------------------------------------------------------------------------------------------
# a whole decode step, as the CPU baseline times it
# ----------------------------------------------------------------------------------------------

def decode_step(pk: PhasorKeyOracle, q: torch.Tensor, ph_q: torch.Tensor, cache_rows: torch.Tensor,
                V: torch.Tensor, head_dim: int) -> torch.Tensor:
    """absorb + scores + softmax + P.V for one sequence: q [H, d], ph_q [1, h], cache_rows [T, W]
    (fp32 dequantised latent), V [T, n_kv, d] bf16 -> [H, d]."""
    qa = pk.absorb(q[:, None, :], ph_q)[:, 0]
    S = pk.scores(qa, cache_rows)
    return attend(S, V, pk.n_kv, head_dim)
