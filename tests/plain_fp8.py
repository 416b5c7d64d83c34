"""Block-scaled 8-bit values and their products in 64 bits: the plain statement that the kernels are compared with."""
import torch

F64 = torch.float64
BLOCK = 128


def blocks(n):
    return (n + BLOCK - 1) // BLOCK


def rows_of(q, scale):
    """``[M, K]`` e4m3 with ``scale [blocks, M]`` as the 64-bit numbers it stands for."""
    col = torch.arange(q.shape[1], device=q.device) // BLOCK
    return q.to(F64) * scale.to(F64).t()[:, col]


def weight_of(q, scale):
    """``[..., N, K]`` e4m3 with ``scale [..., blocks, blocks]`` as the 64-bit numbers it stands for."""
    row, col = (torch.arange(n, device=q.device) // BLOCK for n in q.shape[-2:])
    return q.to(F64) * scale.to(F64)[..., row, :][..., col]


def half_step(x):
    """How far the nearest e4m3 value may be from ``x`` (|x| <= 448): 2^-4 of its magnitude's power of two, at least half of
    the smallest step, 2^-10."""
    return torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6)))) * 2.0 ** -4


def product(a, a_scale, w, w_scale, offsets=None):
    """``(C, S)``: the product in 64 bits and the sums of magnitudes that its rounding errors go by.  Rows behind the last
    expert are NaN."""
    A, W = rows_of(a, a_scale), weight_of(w, w_scale)
    if offsets is None:
        return A @ W.t(), A.abs() @ W.abs().t()
    C = torch.full((A.shape[0], W.shape[1]), float("nan"), dtype=F64, device=A.device)
    S = C.clone()
    o = offsets.tolist()
    for e in range(W.shape[0]):
        C[o[e]:o[e + 1]] = A[o[e]:o[e + 1]] @ W[e].t()
        S[o[e]:o[e + 1]] = A[o[e]:o[e + 1]].abs() @ W[e].abs().t()
    return C, S


def product_error(K, S):
    """A bound on the float32 product's error: every product of two e4m3 values is exact; a block's 128 are added in at most
    128 steps that may cut off a bit each (2^-23), the blocks with a rounding each, and the two scales' product and its
    use with one each (2^-24)."""
    return (2 * min(K, BLOCK) + blocks(K) + 4) * 2.0 ** -24 * S


def swiglu_and_error(C, S, K, s):
    """``(h, bound)`` of ``silu(s g) * (s u)`` from a gate|up product: silu's slope is at most 1.1 and silu(g) at most |g|;
    the exponential's argument is rounded (|g| 2^-23 of the result), the exponential, the reciprocal and the products have
    at most 2^-21 together."""
    I = C.shape[1] // 2
    e = product_error(K, S) * s.abs() + C.abs() * s.abs() * 2.0 ** -23
    g, u = C[:, :I] * s, C[:, I:] * s
    h = g * torch.sigmoid(g) * u
    return h, 1.1 * e[:, :I] * u.abs() + g.abs() * e[:, I:] + 1.1 * e[:, :I] * e[:, I:] + h.abs() * (4 + g.abs()) * 2.0 ** -22
