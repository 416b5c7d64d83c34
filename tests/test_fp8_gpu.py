"""The block-scaled 8-bit operators against a plain statement in 64 bits (needs a GPU)."""
import pytest
import torch

from plain_fp8 import BLOCK, F64, blocks, half_step, product, product_error, rows_of, swiglu_and_error, weight_of

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
E4M3, BF16, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from sharpinference_b200.kernels import ops as _ops
    yield _ops
    _ops.check_status(DEV)


def rnd(*shape, dtype=F32, scale=1.0, seed=0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def rows_definition(x):
    """The definition in the operations and the precision that it is given in."""
    M, K = x.shape
    b = torch.nn.functional.pad(x.float(), (0, blocks(K) * BLOCK - K)).view(M, -1, BLOCK)
    scale = (b.abs().amax(2) * (1.0 / 448.0)).clamp_min(2.0 ** -126)
    q = (b * (1.0 / scale).unsqueeze(2)).to(E4M3).float().view(M, -1)[:, :K]
    return q, scale.t()


def same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=1e30), torch.nan_to_num(b.float(), nan=1e30))


# ---- quantisation -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 5120), (2, 127), (3, 128), (4, 129), (5, 2047), (33, 640), (130, 1000), (1, 16), (7, 8200)])
def test_rows(ops, dtype, M, K):
    x = rnd(M, K, dtype=dtype, scale=3.0, seed=M + K)
    x[0, : K // 2] *= 1e-3
    q, scale = ops.fp8_rows(x)
    assert q.dtype == E4M3 and tuple(q.shape) == (M, K) and tuple(scale.shape) == (blocks(K), M) and q.stride(0) % 16 == 0
    want_q, want_scale = rows_definition(x)
    assert same(q, want_q) and torch.equal(scale, want_scale)
    # and in 64 bits: the scale has two roundings, the quotient two more before the one to e4m3
    x64 = x.to(F64)
    for b in range(blocks(K)):
        amax = x64[:, b * BLOCK:(b + 1) * BLOCK].abs().amax(1)
        assert ((scale[b].to(F64) - amax / 448).abs() <= amax / 448 * 2.0 ** -23 + 2.0 ** -126).all()
    s = scale.to(F64).t()[:, torch.arange(K, device=DEV) // BLOCK]
    v = x64 / s
    assert ((q.to(F64) - v).abs() <= half_step(v) + v.abs() * 2.0 ** -22).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K", [(1400, 5120), (5500, 1003), (10007, 640), (11001, 520), (42000, 130)])
def test_many_rows(ops, dtype, M, K):
    """More than the 9 MB up to which a warp has one row at a time; row counts that are no multiple of what it has then."""
    base = rnd(M, K + 5, dtype=dtype, scale=3.0, seed=K)
    for x in (base[:, :K].contiguous(), base[:, 3:K + 3]):
        q, scale = ops.fp8_rows(x)
        want_q, want_scale = rows_definition(x)
        assert same(q, want_q) and torch.equal(scale, want_scale)
    at = torch.randperm(M, generator=torch.Generator().manual_seed(1))[: M - 3].to(torch.int32).to(DEV)
    q, scale = ops.fp8_rows(base[:, :K], rows=at)
    want_q, want_scale = rows_definition(base[at.long(), :K])
    assert same(q, want_q) and torch.equal(scale, want_scale)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_zeros_tiny_and_broken_numbers(ops, dtype):
    x = rnd(8, 384, dtype=dtype, seed=5)
    x[0] = 0.0
    x[1] = 1e-38
    x[2, 5] = float("nan")
    x[3, 130] = float("inf")
    x[4, 383] = float("-inf")
    x[5] = torch.finfo(dtype).max
    x[6] = -x[6].abs()
    q, scale = ops.fp8_rows(x)
    want_q, want_scale = rows_definition(x)
    assert same(scale, want_scale)
    v = rows_of(q, scale)
    assert torch.equal(v[0], torch.zeros_like(v[0])) and torch.isfinite(v[5]).all()
    bad = torch.zeros(8, 384, dtype=torch.bool, device=DEV)
    bad[2, :128] = bad[3, 128:256] = bad[4, 256:] = True          # a block that holds such a number is NaN, no other is
    assert torch.equal(torch.isnan(v), bad)
    assert same(q[~bad], want_q[~bad])


def test_rows_gathered_strided_and_unaligned(ops):
    wide = rnd(50, 700, dtype=BF16, seed=6)
    rows = torch.tensor([49, 0, 7, 7, 12], dtype=torch.int32, device=DEV)
    for x in (wide, wide[:, 8:400], wide[:, 3:400], wide[::2][:20], wide.float()[:, 1:131]):
        idx = rows % x.shape[0]
        q, scale = ops.fp8_rows(x, rows=idx)
        want_q, want_scale = rows_definition(x[idx.long()])
        assert same(q, want_q) and torch.equal(scale, want_scale)
    q, scale = ops.fp8_rows(wide, rows=rows[:0])
    assert tuple(q.shape) == (0, 700) and tuple(scale.shape) == (6, 0)
    q, scale = ops.fp8_rows(wide[:0])
    assert tuple(q.shape) == (0, 700)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 1), (128, 128), (129, 127), (300, 5000), (3, 130, 260), (2, 127, 16), (5, 1, 300)])
def test_weight(ops, dtype, shape):
    w = rnd(*shape, dtype=dtype, scale=0.02, seed=sum(shape))
    q, scale = ops.fp8_weight(w)
    N, K = shape[-2:]
    assert tuple(q.shape) == shape and tuple(scale.shape) == (*shape[:-2], blocks(N), blocks(K))
    flat, fq, fs = w.reshape(-1, N, K), q.to(F64).reshape(-1, N, K), scale.reshape(-1, blocks(N), blocks(K))
    for e in range(flat.shape[0]):
        for i in range(blocks(N)):
            for j in range(blocks(K)):
                part = (e, slice(i * BLOCK, (i + 1) * BLOCK), slice(j * BLOCK, (j + 1) * BLOCK))
                s = (flat[part].float().abs().amax() * (1.0 / 448.0)).clamp_min(2.0 ** -126)
                assert torch.equal(fs[e, i, j], s)
                v = flat[part].to(F64) / s.to(F64)
                assert ((fq[part] - v).abs() <= half_step(v) + v.abs() * 2.0 ** -22).all()


def test_weight_strided_and_unaligned(ops):
    big = rnd(4, 300, 520, seed=9)
    for w in (big[:, :200, :256], big[:, 3:203, 1:300], big[1, :, 5:], big[::2, :, :128]):
        q, scale = ops.fp8_weight(w)
        want_q, want_scale = ops.fp8_weight(w.contiguous())
        assert same(q, want_q) and torch.equal(scale, want_scale)


# ---- products ---------------------------------------------------------------------------------------------------
def operands(ops, M, N, K, E=None, seed=0):
    a = ops.fp8_rows(rnd(M, K, scale=2.0, seed=seed))
    w = ops.fp8_weight(rnd(*((N, K) if E is None else (E, N, K)), scale=0.05, seed=seed + 1))
    return (*a, *w)


def close(got, want, bound):
    if got.dtype == BF16:
        bound = bound + want.abs() * 2.0 ** -8          # one rounding by half a step
    bad = ~((got.to(F64) - want).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} beyond, worst {float(((got.to(F64) - want).abs() / bound.clamp_min(1e-300)).max()):.3g} of the bound"


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 7168, 5120), (1, 200, 130), (2, 129, 15), (16, 1000, 2048), (17, 256, 127), (33, 520, 4100),
                                   (64, 640, 640), (127, 384, 128), (128, 128, 256), (129, 257, 1000), (300, 1100, 384), (1000, 700, 2500),
                                   (2500, 1300, 513)])
def test_dense(ops, out_dtype, M, N, K):
    t = operands(ops, M, N, K, seed=M + N + K)
    got = ops.fp8_dense(*t, out_dtype=out_dtype)
    want, S = product(*t)
    assert got.dtype == out_dtype and tuple(got.shape) == (M, N)
    close(got, want, product_error(K, S))


def test_dense_bias_out_and_accumulate(ops):
    M, N, K = 70, 333, 700
    t = operands(ops, M, N, K, seed=3)
    want, S = product(*t)
    bias, base = rnd(N, seed=8), rnd(M, N, seed=9)
    err = product_error(K, S) + (want.abs() + bias.abs().to(F64)) * 2.0 ** -24
    close(ops.fp8_dense(*t, bias=bias), want + bias.to(F64), err)
    close(ops.fp8_dense(*t, bias=bias, out_dtype=BF16), want + bias.to(F64), err)
    out = torch.full((M + 3, N), 7.0, device=DEV)
    assert ops.fp8_dense(*t, out=out) is out
    assert (out[M:] == 7.0).all()
    plain = out[:M].clone()
    y = base.clone()
    ops.fp8_dense(*t, out=y, accumulate=True)
    assert torch.equal(y, base + plain)                 # one addition an element


def test_dense_of_no_rows_or_columns(ops):
    t = operands(ops, 4, 130, 64)
    empty = ops.fp8_dense(t[0][:0], t[1][:, :0].contiguous(), t[2], t[3])
    assert tuple(empty.shape) == (0, 130)
    none = ops.fp8_dense(t[0], t[1], t[2][:0], t[3][:0])
    assert tuple(none.shape) == (4, 0)


def test_dense_reads_rows_that_lie_apart(ops):
    M, N, K = 40, 300, 272
    t = operands(ops, M, N, K, seed=4)
    want = ops.fp8_dense(*t)
    wide_a = torch.full((M, 512), 1.0, device=DEV).to(E4M3)
    wide_w = torch.full((N, 400), 1.0, device=DEV).to(E4M3)
    wide_a[:, 16:16 + K] = t[0]
    wide_w[:, 32:32 + K] = t[2]
    assert torch.equal(ops.fp8_dense(wide_a[:, 16:16 + K], t[1], wide_w[:, 32:32 + K], t[3]), want)


def test_dense_broken_numbers_stay_in_their_row(ops):
    M, N, K = 20, 260, 640
    x, w = rnd(M, K, seed=1), rnd(N, K, scale=0.05, seed=2)
    x[3, 200] = float("nan")
    x[11, 5] = float("inf")
    w[256, 639] = float("nan")
    a, b = ops.fp8_rows(x), ops.fp8_weight(w)
    got = ops.fp8_dense(*a, *b)
    bad = torch.zeros(M, N, dtype=torch.bool, device=DEV)
    bad[3] = bad[11] = True
    bad[:, 256:] = True                                 # the weight's block of 128 rows
    assert torch.equal(torch.isnan(got), bad)


OFFSETS = {
    "even": [0, 10, 20, 30, 40], "empty_experts": [0, 0, 37, 37, 40], "one_takes_all": [0, 0, 0, 300, 300],
    "over_a_tile": [0, 129, 130, 300, 555], "none": [0, 0, 0, 0, 0], "rows_behind": [0, 5, 9, 9, 30],
}


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("name", sorted(OFFSETS))
@pytest.mark.parametrize("N,K", [(300, 200), (256, 1024)])
def test_grouped(ops, out_dtype, name, N, K):
    offsets = torch.tensor(OFFSETS[name], dtype=torch.int32, device=DEV)
    last = OFFSETS[name][-1]
    rows = last + (11 if name in ("rows_behind", "none") else 0)
    t = operands(ops, rows, N, K, E=4, seed=rows)
    want, S = product(*t, offsets)
    out = torch.full((rows, N), 5.0, dtype=out_dtype, device=DEV)
    ops.fp8_grouped(*t, offsets, out=out)
    close(out[:last], want[:last], product_error(K, S)[:last])
    assert (out[last:] == 5.0).all()                    # rows of no expert are left as they were
    # weighted, and sent to other places
    to = torch.randperm(rows + 4, generator=torch.Generator().manual_seed(1))[:rows].to(torch.int32).to(DEV)
    weight = rnd(rows + 4, seed=2)
    out = torch.full((rows + 4, N), 5.0, dtype=out_dtype, device=DEV)
    ops.fp8_grouped(*t, offsets, out=out, out_rows=to, row_scale=weight, scale_rows=to)
    there = to[:last].long()
    s = weight[there].to(F64).unsqueeze(1)
    close(out[there], want[:last] * s, (product_error(K, S)[:last] + want[:last].abs() * 2.0 ** -24) * s.abs())
    left = torch.ones(rows + 4, dtype=torch.bool, device=DEV)
    left[there] = False
    assert (out[left] == 5.0).all()
    if out_dtype == F32:
        out2 = torch.full((rows + 4, N), 1.0, device=DEV)
        ops.fp8_grouped(*t, offsets, out=out2, out_rows=to, row_scale=weight, scale_rows=to, accumulate=True)
        assert torch.equal(out2[there], out[there] + 1.0) and (out2[left] == 1.0).all()


@pytest.mark.parametrize("E", [1, 33, 200])
def test_grouped_of_many_experts(ops, E):
    N, K = 130, 144
    counts = torch.randint(0, 4, (E,), generator=torch.Generator().manual_seed(E))
    offsets = torch.zeros(E + 1, dtype=torch.int32)
    offsets[1:] = counts.cumsum(0)
    rows = int(offsets[-1])
    offsets = offsets.to(DEV)
    if rows == 0:
        rows, offsets = 2, torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    t = operands(ops, rows, N, K, E=E, seed=E)
    want, S = product(*t, offsets)
    close(ops.fp8_grouped(*t, offsets), want, product_error(K, S))


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("name", ["even", "empty_experts", "over_a_tile", "rows_behind"])
@pytest.mark.parametrize("I,K", [(128, 200), (384, 1024), (100, 320), (192, 130)])
def test_swiglu(ops, name, I, K, weighted):
    offsets = torch.tensor(OFFSETS[name], dtype=torch.int32, device=DEV)
    last = OFFSETS[name][-1]
    rows = last + (11 if name == "rows_behind" else 0)
    t = operands(ops, rows, 2 * I, K, E=4, seed=I + rows)
    at = torch.randperm(rows, generator=torch.Generator().manual_seed(3)).to(torch.int32).to(DEV) if weighted else None
    weight = rnd(rows, seed=4).abs() if weighted else None
    q, scale = ops.fp8_swiglu(*t, offsets, row_scale=weight, scale_rows=at)
    check_swiglu(q[:last], scale[:, :last], *[v[:last] for v in product(*t, offsets)], K,
                 weight[at.long()][:last].to(F64).unsqueeze(1) if weighted else torch.ones(1, 1, dtype=F64, device=DEV))


def check_swiglu(q, scale, C, S, K, s):
    h, e = swiglu_and_error(C, S, K, s)
    I = h.shape[1]
    assert q.dtype == E4M3 and tuple(q.shape) == (h.shape[0], I) and tuple(scale.shape) == (blocks(I), h.shape[0])
    s64 = scale.to(F64).t()
    for b in range(blocks(I)):
        part = slice(b * BLOCK, (b + 1) * BLOCK)
        amax = h[:, part].abs().amax(1)
        assert ((s64[:, b] - amax / 448).abs() <= amax / 448 * 2.0 ** -23 + e[:, part].amax(1) / 448).all()
    full = s64[:, torch.arange(I, device=DEV) // BLOCK]
    v = h / full
    close(rows_of(q, scale), h, full * (half_step(v.clamp(-448, 448)) * 1.0001 + v.abs() * 2.0 ** -22) + 2 * e)


@pytest.mark.parametrize("M", [1, 100, 129])
@pytest.mark.parametrize("I", [256, 72])
def test_swiglu_dense(ops, M, I):
    t = operands(ops, M, 2 * I, 520, seed=M)
    check_swiglu(*ops.fp8_swiglu(*t), *product(*t), 520, torch.ones(1, 1, dtype=F64, device=DEV))


@pytest.mark.parametrize("split", [1, 2])
def test_silu_of_known_gates(ops, split):
    """Every block of h is one number, silu of a float32 that the product has exactly, so the block's scale shows silu's error: the
    exponential 2^-22, the reciprocal and the two sums 2^-22 together, the products and 1 / 448 another 2^-22."""
    g = torch.cat([torch.linspace(-82, 82, 83), torch.tensor([1e-3, -1e-3, 0.3, 1.0 / 3])]).to(F32)
    n = g.numel()
    a, w = ops.fp8_empty((3, 256), DEV), ops.fp8_empty((2 * n * BLOCK, 256), DEV)
    a.view(torch.uint8).zero_()
    w.view(torch.uint8).zero_()
    a[:, 0] = torch.ones(3, device=DEV).to(E4M3)
    w[:, 0] = torch.ones(2 * n * BLOCK, device=DEV).to(E4M3)
    a_scale, w_scale = torch.ones(2, 3, device=DEV), torch.ones(2 * n, 2, device=DEV)
    w_scale[:n] = g.to(DEV).unsqueeze(1)
    q, scale = ops.fp8_empty((3, n * BLOCK), DEV), torch.empty(n, 3, device=DEV)
    ops._fp8_product(a, a_scale, w, w_scale, None, swiglu=True, out=q, out_scale=scale, split=split)
    h = g.to(F64) * torch.sigmoid(g.to(F64))
    least = 448 * 2.0 ** -126                           # the smallest scale, which a block of zeros has (the gate 0: 448 * 2^-126 - 0)
    assert ((scale.to(F64).cpu() * 448 - h.abs().unsqueeze(1)).abs() <= h.abs().unsqueeze(1) * 3 * 2.0 ** -22 + least * (h == 0).unsqueeze(1)).all()
    assert (q.to(F64).cpu().abs() == 448 * (h != 0).repeat_interleave(BLOCK)).all()


def ragged(rows_up_to, E, seed):
    """Offsets of experts with no, a few, and many rows: tiles whose last warps have no rows before and behind full ones."""
    g = torch.Generator().manual_seed(seed)
    counts = torch.randint(1, rows_up_to, (E,), generator=g)
    counts[torch.randperm(E, generator=g)[: E // 5]] = 0
    counts[torch.randperm(E, generator=g)[: E // 3]] = torch.randint(1, 32, (E // 3,), generator=g)
    offsets = torch.zeros(E + 1, dtype=torch.int32)
    offsets[1:] = counts.cumsum(0)
    return offsets.to(DEV), int(offsets[-1])


# hundreds of tiles more than the GPU has SMs, so that a CTA walks several: blocks of K odd and even in number, one alone; rows of C
# that start on 32 bytes, 16 and fewer
@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("M,N,K", [(2700, 5200, 300), (2689, 5203, 512), (2561, 5128, 100), (5000, 2600, 1000)])
def test_dense_walk_over_many_tiles(ops, out_dtype, M, N, K):
    t = operands(ops, M, N, K, seed=M)
    want, S = product(*t)
    close(ops._fp8_product(*t, None, split=1, out_dtype=out_dtype), want, product_error(K, S))


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("E,N,K,most", [(60, 1040, 384, 200), (90, 1033, 520, 150), (40, 2072, 128, 600)])
def test_grouped_walk_over_many_tiles(ops, out_dtype, E, N, K, most):
    offsets, rows = ragged(most, E, seed=E)
    assert rows > E and (N + 255) // 256 * int(((offsets.diff() + 127) // 128).sum()) > 2 * 148
    t = operands(ops, rows, N, K, E=E, seed=E)
    want, S = product(*t, offsets)
    to = torch.randperm(rows + 9, generator=torch.Generator().manual_seed(1))[:rows].to(torch.int32).to(DEV)
    weight = rnd(rows + 9, seed=2)
    out = torch.full((rows + 9, N), 5.0, dtype=out_dtype, device=DEV)
    ops._fp8_product(*t, offsets, split=1, out=out, out_rows=to, row_scale=weight, scale_rows=to)
    s = weight[to.long()].to(F64).unsqueeze(1)
    close(out[to.long()], want * s, (product_error(K, S) + want.abs() * 2.0 ** -24) * s.abs())
    left = torch.ones(rows + 9, dtype=torch.bool, device=DEV)
    left[to.long()] = False
    assert (out[left] == 5.0).all()


@pytest.mark.parametrize("E,I,K,most", [(40, 1280, 256, 300), (60, 768, 392, 200), (30, 2048, 100, 500)])
def test_swiglu_walk_over_many_tiles(ops, E, I, K, most):
    offsets, rows = ragged(most, E, seed=E + 1)
    assert I // 128 * int(((offsets.diff() + 127) // 128).sum()) > 2 * 148
    t = operands(ops, rows, 2 * I, K, E=E, seed=E)
    weight = rnd(rows, seed=4).abs()
    q, scale = ops.fp8_empty((rows, I), DEV), torch.empty(blocks(I), rows, device=DEV)
    ops._fp8_product(*t, offsets, swiglu=True, out=q, out_scale=scale, row_scale=weight, split=1)
    check_swiglu(q, scale, *product(*t, offsets), K, weight.to(F64).unsqueeze(1))


def test_a_row_does_not_depend_on_the_rest(ops):
    """A row's bits are the same alone and among others of its kind of step, as in the other tensor-core kernels."""
    N, K = 512, 1024
    x = rnd(300, K, seed=1)
    w = ops.fp8_weight(rnd(N, K, scale=0.05, seed=2))
    whole = ops.fp8_dense(*ops.fp8_rows(x), *w)
    part = ops.fp8_dense(*ops.fp8_rows(x[130:300]), *w)
    assert torch.equal(whole[130:], part)
    q, s = ops.fp8_swiglu(*ops.fp8_rows(x), *w)
    q1, s1 = ops.fp8_swiglu(*ops.fp8_rows(x[130:300]), *w)
    assert same(q[130:], q1) and torch.equal(s[:, 130:], s1)


def mixture(ops, x, expert, weight, gate_up, down):
    """A mixture's experts as they would be used: rows sorted by expert, quantised, both products, weighted sum."""
    T, k = expert.shape
    E = gate_up[0].shape[0]
    offsets, pairs = ops.moe_sort(expert.view(-1), E)
    a = ops.fp8_rows(x, rows=ops.moe_pair_tokens(pairs, k))
    h = ops.fp8_swiglu(*a, *gate_up, offsets)
    y = ops.fp8_grouped(*h, *down, offsets, out_rows=pairs, row_scale=weight.view(-1), scale_rows=pairs)
    return ops.moe_combine(y, k), (offsets, pairs, a, h)


def mixture_case(ops, T, k, E, H, I, seed):
    x = rnd(T, H, dtype=BF16, seed=seed)
    router = rnd(E, H, scale=H ** -0.5, seed=seed + 1)
    expert, weight, _ = ops.router_topk(x.float(), router, k, renormalize=True)
    return x, expert, weight, ops.fp8_weight(rnd(E, 2 * I, H, scale=H ** -0.5, seed=seed + 2)), ops.fp8_weight(rnd(E, H, I, scale=I ** -0.5, seed=seed + 3))


@pytest.mark.parametrize("T,k,E,H,I", [(1, 2, 8, 256, 128), (19, 3, 8, 320, 200), (300, 2, 4, 512, 384)])
def test_together(ops, T, k, E, H, I):
    case = mixture_case(ops, T, k, E, H, I, seed=T)
    x, expert, weight, gate_up, down = case
    got, (offsets, pairs, a, h) = mixture(ops, *case)
    # every stage from the stage before it
    want_q, want_scale = rows_definition(x[(pairs // k).long()])
    assert same(a[0], want_q) and torch.equal(a[1], want_scale)
    check_swiglu(*h, *product(*a, *gate_up, offsets), H, torch.ones(1, 1, dtype=F64, device=DEV))
    C, S = product(*h, *down, offsets)
    w = weight.view(-1)[pairs.long()].to(F64).unsqueeze(1)
    y, bound = torch.zeros(T * k, H, dtype=F64, device=DEV), torch.zeros(T * k, H, dtype=F64, device=DEV)
    y[pairs.long()] = C * w
    bound[pairs.long()] = (product_error(I, S) + C.abs() * 2.0 ** -24) * w
    total = y.view(T, k, H)
    close(got, total.sum(1), bound.view(T, k, H).sum(1) + k * 2.0 ** -24 * total.abs().sum(1))


def test_in_a_graph_and_on_another_stream(ops):
    case = mixture_case(ops, 5, 2, 8, 256, 256, seed=11)
    want, _ = mixture(ops, *case)
    x = case[0].clone()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):                                  # two graphs of the same work, replayed side by side
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mixture(ops, x, *case[1:])[0])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    x.copy_(rnd(5, 256, dtype=BF16, seed=99))           # new inputs, the same graph
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], mixture(ops, x, *case[1:])[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = mixture(ops, *case)
    side.synchronize()
    assert torch.equal(got, want)


def test_the_first_call_of_a_process_captured(ops, monkeypatch):
    """The status word that a captured call brings into being is zero at once and is no part of the graph: a replay does not take
    back what a kernel has recorded."""
    t = operands(ops, 3, 200, 300)
    want = ops.fp8_dense(*t)
    torch.cuda.synchronize()
    monkeypatch.setattr(ops, "_status_words", {})
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.fp8_dense(*t)
    word = ops.status_word(DEV)
    ops.check_status(DEV)
    g.replay()
    word.fill_(8)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    with pytest.raises(ops.KernelError, match="code 8"):
        ops.check_status(DEV)
    ops.check_status(DEV)


@pytest.mark.parametrize("split", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("M,N,K", [(1, 300, 1024), (37, 256, 1100), (128, 130, 1153), (200, 515, 2048)])
def test_split_over_k(ops, split, M, N, K):
    """Every way of cutting K over the CTAs of a cluster, whatever the sizes would choose."""
    t = operands(ops, M, N, K, seed=M + split)
    want, S = product(*t)
    bias, base = rnd(N, seed=8), rnd(M, N, seed=9)
    err = product_error(K, S) + split * 2.0 ** -24 * S
    close(ops._fp8_product(*t, None, split=split), want, err)
    close(ops._fp8_product(*t, None, split=split, bias=bias, out_dtype=BF16), want + bias.to(F64), err + (want.abs() + bias.abs()) * 2.0 ** -24)
    out = base.clone()
    ops._fp8_product(*t, None, split=split, out=out, accumulate=True)
    close(out, want + base.to(F64), err + (want.abs() + base.abs()) * 2.0 ** -23)


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("start", [0, 8, 4, 1])
@pytest.mark.parametrize("N", [272, 264, 260, 261, 24, 4])
def test_outputs_on_every_boundary(ops, N, start, out_dtype):
    """Rows of the output that start on 32, 16 or fewer bytes, few and many of them; what lies around them stays."""
    K = 200
    for M in (3, 41, 140):
        t = operands(ops, M, N, K, seed=M + N)
        want, S = product(*t)
        around = torch.full((start + M * N + 64,), 7.0, dtype=out_dtype, device=DEV)
        out = around[start:start + M * N].view(M, N)
        ops._fp8_product(*t, None, split=1, out=out)
        close(out, want, product_error(K, S))
        assert (around[:start] == 7.0).all() and (around[start + M * N:] == 7.0).all()
        if out_dtype == F32:
            plain = out.clone()
            ops._fp8_product(*t, None, split=1, out=out, accumulate=True)
            assert torch.equal(out, plain + plain)


@pytest.mark.parametrize("split", [1, 3, 8])
@pytest.mark.parametrize("name", ["empty_experts", "over_a_tile", "rows_behind"])
def test_split_over_k_by_experts(ops, name, split):
    offsets = torch.tensor(OFFSETS[name], dtype=torch.int32, device=DEV)
    last, I, K, N = OFFSETS[name][-1], 256, 1030, 300
    rows = last + (11 if name == "rows_behind" else 0)
    at = torch.randperm(rows, generator=torch.Generator().manual_seed(3)).to(torch.int32).to(DEV)
    weight = rnd(rows, seed=4).abs()
    s = weight[at.long()][:last].to(F64).unsqueeze(1)
    t = operands(ops, rows, 2 * I, K, E=4, seed=I + rows)
    q, scale = ops.fp8_empty((rows, I), DEV), torch.empty(blocks(I), rows, device=DEV)
    ops._fp8_product(*t, offsets, swiglu=True, out=q, out_scale=scale, row_scale=weight, scale_rows=at, split=split)
    C, S = product(*t, offsets)
    check_swiglu(q[:last], scale[:, :last], C[:last], S[:last] * (1 + split * 2.0 ** -9), K, s)
    t = operands(ops, rows, N, K, E=4, seed=rows)
    C, S = product(*t, offsets)
    out = torch.full((rows, N), 5.0, device=DEV)
    ops._fp8_product(*t, offsets, out=out, out_rows=at, row_scale=weight, scale_rows=at, split=split)
    there = at[:last].long()
    close(out[there], C[:last] * s, (product_error(K, S)[:last] + split * 2.0 ** -24 * S[:last] + C[:last].abs() * 2.0 ** -24) * s)
    left = torch.ones(rows, dtype=torch.bool, device=DEV)
    left[there] = False
    assert (out[left] == 5.0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantisation_of_rows_that_start_anywhere(ops, dtype):
    """Every distance of a row's start from a 16-byte boundary, rows that end inside of one, at the end of their memory."""
    step = 16 // torch.tensor([], dtype=dtype).element_size()
    for off in range(step):
        for K in (1, step, 125, 128, 131, 255, 263):
            x = rnd(9, off + K, dtype=dtype, seed=off + K)
            part = x[:, off:]                                  # ends where its memory ends
            q, scale = ops.fp8_rows(part)
            want_q, want_scale = rows_definition(part)
            assert same(q, want_q) and torch.equal(scale, want_scale)
            q, scale = ops.fp8_weight(part)
            want_q, want_scale = ops.fp8_weight(torch.nn.functional.pad(part, (0, -K % 16))[:, :K])
            assert same(q, want_q) and torch.equal(scale, want_scale)


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("split", [1, 3])
def test_a_wait_that_runs_out_is_reported_and_the_kernel_returns(ops, split, swiglu):
    """One launch loads nothing behind the first block of K and polls each wait a few thousand times: a wait runs out, the kernel
    records a code and returns (no fault, no hang), check_status raises it, and the next launch is right again."""
    M, I, K = 300, 256, 1100
    t = operands(ops, M, 2 * I, K, seed=M)

    def product_of():
        out = ops.fp8_empty((M, I), DEV) if swiglu else torch.empty(M, 2 * I, device=DEV)
        scale = torch.empty(blocks(I), M, device=DEV)
        ops._fp8_product(*t, None, split=split, out=out, **(dict(swiglu=True, out_scale=scale) if swiglu else {}))
        return out, scale

    want = product_of()
    ops.check_status(DEV)
    ops.fp8_set_wait_test()
    product_of()
    with pytest.raises(ops.KernelError, match="gave up"):
        ops.check_status(DEV)
    ops.check_status(DEV)                               # the word is back at zero
    got = product_of()
    ops.check_status(DEV)
    assert same(got[0], want[0]) and (not swiglu or torch.equal(got[1], want[1]))
