"""The mixture layer for a few tokens against a plain statement in 64 bits (needs a GPU)."""
import pytest
import torch

from plain_fp8 import F64, weight_of

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from sharpinference_b200.kernels import ops as _ops
    yield _ops
    _ops.check_status(DEV)


def rnd(*shape, dtype=F32, scale=1.0, seed=0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def layer(ops, T, E, H, I, weights="bfloat16", seed=0):
    h32 = rnd(T, H, scale=1.5, seed=seed)
    c = {"h": h32.to(BF16), "h32": h32, "router": rnd(E, H, scale=H ** -0.5, seed=seed + 1)}
    gate_up, down = rnd(E, 2 * I, H, scale=H ** -0.5, seed=seed + 2), rnd(E, H, I, scale=I ** -0.5, seed=seed + 3)
    if weights == "e4m3":
        c["gate_up"], c["gate_up_scale"] = ops.fp8_weight(gate_up)
        c["down"], c["down_scale"] = ops.fp8_weight(down)
    else:
        c["gate_up"], c["down"], c["gate_up_scale"], c["down_scale"] = gate_up.to(BF16), down.to(BF16), None, None
    return c


def call(ops, c, k, **more):
    return ops.moe_few(c["h"], c["router"], c["gate_up"], c["down"], k, h32=c["h32"], gate_up_scale=c["gate_up_scale"],
                       down_scale=c["down_scale"], **more)


def plain(c, expert, weight, on, act_step=2.0 ** -16):
    """``(y, bound)``: the layer in 64 bits under the given choices, and a bound on the kernel's error: float32 sums of n
    terms (n 2^-24 of the sum of magnitudes at most), silu's slope at most 1.1, act rounded to two bfloat16 (2^-16) or, with 8-bit weights, to
    float16 (2^-11; below 2^-14 of a block's scale 2^-25 of it, where the block's largest is 2^14 to 2^15 of it)."""
    h = c["h"].to(F64)
    T, H = h.shape
    y, bound = torch.zeros_like(h), torch.zeros_like(h)
    W = {n: c[n].to(F64) if c[n + "_scale"] is None else weight_of(c[n], c[n + "_scale"]) for n in ("gate_up", "down")}
    I = W["down"].shape[2]
    for t in range(T):
        for e, w in zip(expert[t].tolist(), weight[t].to(F64).tolist()):
            gu = W["gate_up"][e] @ h[t]
            err = (H + 8) * 2.0 ** -24 * (W["gate_up"][e].abs() @ h[t].abs())
            if on == "input":
                gu, err = gu * w, err * abs(w) + gu.abs() * abs(w) * 2.0 ** -24
            g, u = gu[:I], gu[I:]
            act = g * torch.sigmoid(g) * u
            err = 1.1 * err[:I] * u.abs() + g.abs() * err[I:] + act.abs() * (8 + g.abs()) * 2.0 ** -23
            if on == "output":
                act, err = act * w, err * abs(w) + act.abs() * abs(w) * 2.0 ** -24
            if c["down_scale"] is None:
                err = err + act.abs() * act_step
            else:
                err = err + act.abs() * 2.0 ** -11 + act.abs().max() * 2.0 ** -38
            y[t] += W["down"][e] @ act
            bound[t] += W["down"][e].abs() @ (err + (I * expert.shape[1] + 40) * 2.0 ** -24 * act.abs())
    return y, bound


def close(got, want, bound):
    if got.dtype == BF16:
        bound = bound + (want.abs() + bound) * 2.0 ** -8
    bad = ~((got.to(F64) - want).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} beyond, worst {float(((got.to(F64) - want).abs() / bound.clamp_min(1e-300)).max()):.3g} of the bound"


@pytest.mark.parametrize("weights", ["bfloat16", "e4m3"])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 2, 128, 64), (1, 128, 8, 2048, 768), (2, 3, 3, 1000, 40), (5, 16, 1, 520, 200), (8, 16, 4, 1024, 512),
                                       (9, 16, 2, 1024, 136), (16, 64, 8, 640, 384), (16, 4, 4, 256, 1000), (16, 300, 32, 128, 64),
                                       (3, 1, 1, 64, 8), (16, 1024, 32, 64, 8), (2, 4, 2, 8, 8), (16, 2, 1, 9008, 64), (13, 4, 2, 64, 2504)])
def test_layer(ops, weights, T, E, k, H, I):
    c = layer(ops, T, E, H, I, weights, seed=T + E + H)
    for i, on in enumerate(("input", "output")):
        for scoring, renormalize in (("sigmoid", bool(i)), ("softmax_chosen", False)):
            expert, weight, _ = ops.router_topk(c["h32"], c["router"], k, scoring=scoring, renormalize=renormalize, scale=1.3)
            y, bound = plain(c, expert, weight, on)
            got = call(ops, c, k, scoring=scoring, renormalize=renormalize, scale=1.3, weights_on=on)
            assert got.dtype == F32 and tuple(got.shape) == (T, H)
            close(got, y, bound)
    close(call(ops, c, k, scoring="softmax_chosen", scale=1.3, out_dtype=BF16), y, bound)


# widths at which a block of the grid has more than 16 and more than 32 rows of the down matrices, and each of its warps several
# blocks of K of the chosen experts
@pytest.mark.parametrize("weights", ["bfloat16", "e4m3"])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 3, 5120, 1000), (5, 8, 2, 5120, 1048), (12, 8, 3, 5120, 1000), (3, 4, 2, 9008, 1200),
                                       (16, 6, 3, 9000, 1000), (8, 6, 2, 7104, 1304)])
def test_wide_layer(ops, weights, T, E, k, H, I):
    c = layer(ops, T, E, H, I, weights, seed=T + H)
    expert, weight, _ = ops.router_topk(c["h32"], c["router"], k, renormalize=True)
    close(call(ops, c, k, renormalize=True), *plain(c, expert, weight, "output"))


@pytest.mark.parametrize("T,H,I", [(1, 257, 130), (11, 1001, 74), (4, 17, 2)])
def test_odd_widths_of_8_bit_weights(ops, T, H, I):
    c = layer(ops, T, 6, H, I, "e4m3", seed=H)
    expert, weight, _ = ops.router_topk(c["h32"], c["router"], 3)
    close(call(ops, c, 3), *plain(c, expert, weight, "output"))


def test_bias_correction_and_router_without_float32(ops):
    T, E, H, I, k = 7, 12, 256, 128, 3
    c = layer(ops, T, E, H, I, seed=4)
    bias, correction = rnd(E, seed=5), rnd(E, seed=6)
    c["h32"] = None
    expert, weight, _ = ops.router_topk(c["h"].float(), c["router"], k, bias=bias, correction=correction, renormalize=True)
    close(call(ops, c, k, bias=bias, correction=correction, renormalize=True), *plain(c, expert, weight, "output"))


def test_ties_go_to_the_lowest_index(ops):
    T, E, H, I = 3, 40, 128, 64
    c = layer(ops, T, E, H, I, seed=1)
    c["router"].zero_()
    expert = torch.arange(4, device=DEV).repeat(T, 1)
    close(call(ops, c, 4), *plain(c, expert, torch.full((T, 4), 0.5, device=DEV), "output"))


@pytest.mark.parametrize("E", [40, 300])
def test_zeros_of_both_signs_are_a_tie(ops, E):
    """Logits of -0 (products too small for float32 and a bias of -0) and of 0 are equal: the lowest indices are chosen."""
    T, H, I = 3, 128, 64
    c = layer(ops, T, E, H, I, seed=1)
    c["h32"].fill_(1e-30)
    c["router"].fill_(-1e-30)
    c["router"][1::2] = 1e-30
    bias = torch.full((E,), -0.0, device=DEV)
    expert, weight, _ = ops.router_topk(c["h32"], c["router"], 4, scoring="softmax_chosen", bias=bias)
    assert torch.equal(expert, torch.arange(4, device=DEV, dtype=torch.int32).repeat(T, 1))
    close(call(ops, c, 4, scoring="softmax_chosen", bias=bias), *plain(c, expert, weight, "output"))


@pytest.mark.parametrize("E", [12, 300])
def test_softmax_whose_largest_logit_is_not_the_first_choice(ops, E):
    """A correction enters the choice alone: logits far above the first choice's are among the chosen."""
    T, H, I, k = 3, 128, 64, 3
    c = layer(ops, T, E, H, I, seed=3)
    c["router"].zero_()
    bias, correction = torch.zeros(E, device=DEV), torch.zeros(E, device=DEV)
    bias[:4] = torch.tensor([0.0, 200.0, -5.0, 199.0], device=DEV)
    correction[:4] = torch.tensor([2000.0, 1000.0, 0.0, 900.0], device=DEV)
    chosen = torch.tensor([0, 1, 3], dtype=torch.int32, device=DEV)
    weight = torch.softmax(bias[chosen.long()].to(F64), 0)
    expert, got, _ = ops.router_topk(c["h32"], c["router"], k, scoring="softmax_chosen", bias=bias, correction=correction)
    assert torch.equal(expert, chosen.repeat(T, 1))
    assert ((got.to(F64) - weight).abs() <= weight * 2.0 ** -20 + 2.0 ** -126).all()       # (exp(-200) is 0 in float32)
    y = call(ops, c, k, scoring="softmax_chosen", bias=bias, correction=correction)
    want, bound = plain(c, expert, weight.repeat(T, 1), "output")
    close(y, want, bound + want.abs() * 2.0 ** -20)     # the weights: exponentials and a quotient of float32


def test_add_and_out(ops):
    T, E, H, I, k = 4, 8, 256, 128, 2
    c = layer(ops, T, E, H, I, seed=2)
    y = call(ops, c, k)
    base = rnd(T, H, seed=3)
    assert torch.equal(call(ops, c, k, add=base), y + base)
    buf = base.clone()
    assert call(ops, c, k, add=buf, out=buf) is buf
    assert torch.equal(buf, y + base)
    assert tuple(ops.moe_few(c["h"][:0], c["router"], c["gate_up"], c["down"], k).shape) == (0, H)


@pytest.mark.parametrize("weights", ["bfloat16", "e4m3"])
def test_broken_numbers_stay_with_their_token(ops, weights):
    T, E, H, I, k = 6, 8, 256, 128, 2
    c = layer(ops, T, E, H, I, weights, seed=9)
    whole = call(ops, c, k)
    for value in (float("nan"), float("inf")):
        d = dict(c, h=c["h"].clone(), h32=c["h32"].clone())
        d["h"][2, 7] = d["h32"][2, 7] = value
        y = call(ops, d, k)
        assert torch.isnan(y[2]).all()
        others = [0, 1, 3, 4, 5]
        assert torch.isfinite(y[others]).all()
        expert, weight, _ = ops.router_topk(c["h32"], c["router"], k)
        want, bound = plain(c, expert, weight, "output")
        close(y[others], want[others], bound[others])
    assert torch.equal(call(ops, c, k), whole)


@pytest.mark.parametrize("weights,where", [("bfloat16", "element"), ("e4m3", "element"), ("e4m3", "scale")])
@pytest.mark.parametrize("T,H,I", [(6, 256, 136), (13, 264, 128), (8, 5120, 200), (16, 2600, 264)])
def test_broken_weights_stay_with_the_tokens_that_chose_their_expert(ops, weights, T, H, I, where):
    """A NaN or an infinity in one expert's matrix: the other tokens' outputs are the bits that they are with whole weights."""
    E, k = 8, 2
    c = layer(ops, T, E, H, I, weights, seed=T)
    whole = call(ops, c, k)
    expert = ops.router_topk(c["h32"], c["router"], k)[0]
    users = [(expert == e).any(1) for e in range(E)]
    e = next(i for i in range(E) if 0 < int(users[i].sum()) < T)
    mine, others = users[e], ~users[e]
    for name, row in (("down", H - 3), ("down", 17), ("gate_up", I + 5), ("gate_up", 0)):
        for value in (float("nan"), float("inf"), float("-inf")):
            d = dict(c)
            if where == "scale":
                d[name + "_scale"] = c[name + "_scale"].clone()
                d[name + "_scale"][e, row // 128, 0] = value
            elif weights == "e4m3":
                d[name] = ops.fp8_empty(c[name].shape, DEV).copy_(c[name])
                d[name].view(torch.uint8)[e, row, 3] = 0x7f if value > 0 or value != value else 0xff      # e4m3 has NaN of both signs
            else:
                d[name] = c[name].clone()
                d[name][e, row, 3] = value
            y = call(ops, d, k)
            assert torch.equal(y[others], whole[others])
            if name == "down":                          # (one row of the matrix, or a scale's block of them, is one output element)
                at = torch.arange(H, device=DEV)
                hit = at // 128 == row // 128 if where == "scale" else at == row
                assert not torch.isfinite(y[mine][:, hit]).any() and torch.equal(y[mine][:, ~hit], whole[mine][:, ~hit])
            else:
                assert not torch.isfinite(y[mine]).any()


def test_weights_whose_rows_lie_apart(ops):
    T, E, H, I, k = 5, 6, 256, 128, 2
    c = layer(ops, T, E, H, I, seed=12)
    want = call(ops, c, k)
    wide = torch.full((E, 2 * I, H + 24), float("nan"), dtype=BF16, device=DEV)
    wide[..., :H] = c["gate_up"]
    assert torch.equal(call(ops, dict(c, gate_up=wide[..., :H]), k), want)


@pytest.mark.parametrize("H,I", [(257, 130), (128, 64)])
def test_what_lies_between_rows_of_8_bit_weights_is_not_read(ops, H, I):
    T, E, k = 5, 6, 2
    c = layer(ops, T, E, H, I, "e4m3", seed=12)
    want = call(ops, c, k)
    for name in ("gate_up", "down"):
        n, m = c[name].shape[1:]
        wide = torch.full((E, n, (m + 15) // 16 * 16 + 32), 0x7f, dtype=torch.uint8, device=DEV)       # e4m3's NaN
        wide[..., :m] = c[name].view(torch.uint8) if c[name].is_contiguous() else c[name].contiguous().view(torch.uint8)
        c[name] = wide.view(torch.float8_e4m3fn)[..., :m]
    assert torch.equal(call(ops, c, k), want)


@pytest.mark.parametrize("weights", ["bfloat16", "e4m3"])
def test_the_same_again_in_graphs_and_on_streams(ops, weights):
    T, E, H, I, k = 6, 32, 512, 256, 4
    c = layer(ops, T, E, H, I, weights, seed=21)
    want = call(ops, c, k)
    for _ in range(20):
        assert torch.equal(call(ops, c, k), want)
    graphs, outs = [], []
    for _ in range(2):                                  # two graphs of the same layer, replayed side by side
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(ops, c, k))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            side = call(ops, c, k)
    torch.cuda.synchronize()
    assert torch.equal(side, want) and all(torch.equal(o, want) for o in outs)


def test_calls_side_by_side(ops):
    """Layers on streams of two priorities at once, with a product that fills the GPU on a third: each layer's blocks wait for one
    another, none for another launch's."""
    E, k, H, I = 16, 4, 512, 256
    layers = [layer(ops, T, E, H, I, seed=T) for T in (3, 12)]
    want = [call(ops, c, k) for c in layers]
    a, w = ops.fp8_rows(rnd(300, 1024, seed=1)), ops.fp8_weight(rnd(7168, 1024, seed=2))
    product = ops.fp8_dense(*a, *w)
    streams = [torch.cuda.Stream(priority=p) for p in (0, -1, -2)]
    torch.cuda.synchronize()
    got = [[], [], []]
    for i in range(60):
        for j, c in enumerate(layers):
            with torch.cuda.stream(streams[j]):
                got[j].append(call(ops, c, k))
        if i % 3 == 0:
            with torch.cuda.stream(streams[2]):
                got[2].append(ops.fp8_dense(*a, *w))
    torch.cuda.synchronize()
    ops.check_status(DEV)
    assert all(torch.equal(y, want[j]) for j in range(2) for y in got[j]) and all(torch.equal(y, product) for y in got[2])


def test_calls_of_several_threads(ops, monkeypatch):
    """Layers whose kernels take different amounts of shared memory, launched by four threads at once."""
    import threading
    layers = [(layer(ops, 8, 1024, 64, 8, seed=1), 32), (layer(ops, 1, 2, 64, 8, seed=2), 1)]
    want = [call(ops, c, k) for c, k in layers]
    # the launches alone, again and again: a call's arguments, and what it allocated kept alive
    launch, empty, args, kept = ops.kernel("sharpi_moe_few"), torch.empty, [], []
    streams = [torch.cuda.Stream() for _ in range(4)]
    monkeypatch.setattr(torch, "empty", lambda *a, **k: kept.append(empty(*a, **k)) or kept[-1])
    monkeypatch.setattr(ops, "kernel", lambda symbol: lambda *a: args.append(a) or 0)
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            c, k = layers[i % 2]
            got.append(call(ops, c, k))
    monkeypatch.undo()
    torch.cuda.synchronize()
    start, codes = threading.Barrier(4), [set() for _ in streams]

    def work(i):
        start.wait()
        for _ in range(3000):
            codes[i].add(launch(*args[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert codes == [{0}] * 4
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))


def test_beside_the_chain_of_kernels(ops):
    """The same layer as the parts run it: one launch after the other over sorted rows, in bfloat16."""
    T, E, H, I, k = 8, 16, 512, 256, 2
    c = layer(ops, T, E, H, I, seed=30)
    expert, weight, _ = ops.router_topk(c["h32"], c["router"], k)
    offsets, pairs = ops.moe_sort(expert.view(-1), E)
    rows = ops.gather_rows_bf16(c["h"], ops.moe_pair_tokens(pairs, k))
    ones = torch.ones(T * k, device=DEV)
    act = ops.tc_grouped_gemm(rows, c["gate_up"], offsets, mode=ops.TC_MODE_SWIGLU, row_scale=ones)
    y = torch.empty(T * k, H, device=DEV)
    ops.tc_grouped_gemm(act, c["down"], offsets, mode=ops.TC_MODE_STORE, out=y, out_rows=pairs, row_scale=weight.view(-1), scale_rows=pairs)
    chain = ops.moe_combine(y, k)
    want, bound = plain(c, expert, weight, "output")
    close(call(ops, c, k), want, bound)
    close(chain, *plain(c, expert, weight, "output", act_step=2.0 ** -8))      # (that one rounds act to bfloat16)


def test_a_barrier_that_is_not_reached_is_reported(ops):
    """Codes of waits that gave up reach the host through the status word."""
    ops.status_word(DEV).fill_(19)
    with pytest.raises(ops.KernelError, match="19"):
        ops.check_status(DEV)
    ops.check_status(DEV)


@pytest.mark.parametrize("weights", ["bfloat16", "e4m3"])
@pytest.mark.parametrize("T", [3, 12])
def test_a_wait_for_other_blocks_that_runs_out(ops, weights, T):
    """The blocks of one launch poll for one another not once: the kernel records its code and returns, and the next call is right."""
    c = layer(ops, T, 8, 256, 128, weights, seed=T)
    want = call(ops, c, 2)
    ops.check_status(DEV)
    ops.moe_few_set_wait_test(0)
    call(ops, c, 2)
    with pytest.raises(ops.KernelError, match="code 19"):
        ops.check_status(DEV)
    ops.check_status(DEV)                               # the word is back at zero
    assert torch.equal(call(ops, c, 2), want)
    ops.check_status(DEV)
