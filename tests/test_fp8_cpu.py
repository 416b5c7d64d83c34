"""What the block-scaled 8-bit operators and the mixture layer for a few tokens refuse, without a GPU: tensors that say they are on the device, and kernels that
only note that they were called."""
import pytest
import torch

from sharpinference_b200.kernels import ops
from sharpinference_b200.kernels.library import KernelError

E4M3, BF16, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32


class OnDevice(torch.Tensor):
    is_cuda = property(lambda self: True)


def dev(t):
    return t.as_subclass(OnDevice)


@pytest.fixture
def calls(monkeypatch):
    seen = []

    def kernel(symbol):
        def launch(*args):
            seen.append((symbol, args))
            return 0
        return launch

    monkeypatch.setattr(ops, "kernel", kernel)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    monkeypatch.setattr(ops, "sm_count", lambda device=None: 148)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)     # the CPU's index
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: dev(empty(*a, **k)))
    return seen


def operands(M=5, N=300, K=200, E=None):
    shape = (N, K) if E is None else (E, N, K)
    return [dev(ops.fp8_empty((M, K), "cpu")), dev(torch.ones(ops.fp8_blocks(K), M)),
            dev(ops.fp8_empty(shape, "cpu")), dev(torch.ones(*shape[:-2], ops.fp8_blocks(N), ops.fp8_blocks(K)))]


OFFSETS = dev(torch.tensor([0, 2, 2, 5], dtype=torch.int32))


def test_calls_that_are_taken(calls):
    ops.fp8_rows(dev(torch.zeros(5, 200)))
    ops.fp8_rows(dev(torch.zeros(5, 300, dtype=BF16)[:, 7:200]), rows=dev(torch.zeros(9, dtype=torch.int32)))
    ops.fp8_weight(dev(torch.zeros(3, 20, 30)))
    ops.fp8_dense(*operands())
    ops.fp8_dense(*operands(), bias=dev(torch.zeros(300)), out_dtype=BF16)
    ops.fp8_grouped(*operands(E=3), OFFSETS, out_rows=dev(torch.arange(5, dtype=torch.int32)))
    ops.fp8_swiglu(*operands(N=256, E=3), OFFSETS)
    ops.fp8_swiglu(*operands(N=256))
    assert [s for s, _ in calls] == ["sharpi_fp8_rows"] * 2 + ["sharpi_fp8_weight"] + ["sharpi_fp8_gemm"] * 5


def test_swiglu_of_other_widths_is_put_together(calls):
    q, scale = ops.fp8_swiglu(*operands(N=200))
    assert [s for s, _ in calls] == ["sharpi_fp8_gemm", "sharpi_swiglu", "sharpi_fp8_rows"]
    assert tuple(q.shape) == (5, 100) and tuple(scale.shape) == (1, 5)


def test_rows_of_8_bit_tensors_start_on_16_bytes():
    for shape in ((3, 1), (3, 16), (2, 3, 17), (4, 100)):
        q = ops.fp8_empty(shape, "cpu")
        assert tuple(q.shape) == shape and q.dtype == E4M3 and q.stride(-2) % 16 == 0 and 0 <= q.stride(-2) - shape[-1] < 16


REFUSED = {
    "rows_on_the_cpu": lambda: ops.fp8_rows(torch.zeros(5, 200)),
    "rows_float16": lambda: ops.fp8_rows(dev(torch.zeros(5, 200, dtype=torch.float16))),
    "rows_3d": lambda: ops.fp8_rows(dev(torch.zeros(5, 4, 200))),
    "rows_of_no_width": lambda: ops.fp8_rows(dev(torch.zeros(5, 0))),
    "rows_columns_apart": lambda: ops.fp8_rows(dev(torch.zeros(200, 5)).t()),
    "rows_index_int64": lambda: ops.fp8_rows(dev(torch.zeros(5, 200)), rows=dev(torch.zeros(5, dtype=torch.int64))),
    "rows_from_none": lambda: ops.fp8_rows(dev(torch.zeros(0, 200)), rows=dev(torch.zeros(5, dtype=torch.int32))),
    "weight_on_the_cpu": lambda: ops.fp8_weight(torch.zeros(5, 200)),
    "weight_1d": lambda: ops.fp8_weight(dev(torch.zeros(200))),
    "weight_transposed": lambda: ops.fp8_weight(dev(torch.zeros(200, 5)).t()),
    "weight_of_no_width": lambda: ops.fp8_weight(dev(torch.zeros(5, 0))),
    "weight_float64": lambda: ops.fp8_weight(dev(torch.zeros(5, 200, dtype=torch.float64))),
    "dense_on_the_cpu": lambda: ops.fp8_dense(*[t.as_subclass(torch.Tensor) for t in operands()]),
    "dense_of_experts": lambda: ops.fp8_dense(*operands(E=3)),
    "dense_inner_sizes": lambda: ops.fp8_dense(*operands(K=200)[:2], *operands(K=184)[2:]),
    "dense_bf16_rows": lambda: ops.fp8_dense(dev(torch.zeros(5, 200, dtype=BF16)), *operands()[1:]),
    "dense_rows_scale_shape": lambda: ops.fp8_dense(operands()[0], dev(torch.ones(5, 2)), *operands()[2:]),
    "dense_rows_scale_dtype": lambda: ops.fp8_dense(operands()[0], dev(torch.ones(2, 5, dtype=BF16)), *operands()[2:]),
    "dense_weight_scale_shape": lambda: ops.fp8_dense(*operands()[:3], dev(torch.ones(2, 3))),
    "dense_unaligned_rows": lambda: ops.fp8_dense(dev(torch.zeros(5, 200, dtype=torch.uint8).view(E4M3)), *operands()[1:]),
    "dense_unaligned_start": lambda: ops.fp8_dense(dev(torch.zeros(5, 208, dtype=torch.uint8).view(E4M3)[:, 8:]), *operands()[1:]),
    "dense_overlapping_rows": lambda: ops.fp8_dense(dev(torch.zeros(1, 400, dtype=torch.uint8).view(E4M3)[:, :200].expand(5, 200)), *operands()[1:]),
    "dense_out_float16": lambda: ops.fp8_dense(*operands(), out_dtype=torch.float16),
    "dense_out_shape": lambda: ops.fp8_dense(*operands(), out=dev(torch.zeros(4, 300))),
    "dense_out_columns": lambda: ops.fp8_dense(*operands(), out=dev(torch.zeros(5, 301))),
    "dense_out_apart": lambda: ops.fp8_dense(*operands(), out=dev(torch.zeros(5, 400))[:, :300]),
    "dense_add_to_nothing": lambda: ops.fp8_dense(*operands(), accumulate=True),
    "dense_add_to_bf16": lambda: ops.fp8_dense(*operands(), out=dev(torch.zeros(5, 300, dtype=BF16)), accumulate=True),
    "dense_bias_size": lambda: ops.fp8_dense(*operands(), bias=dev(torch.zeros(299))),
    "dense_bias_dtype": lambda: ops.fp8_dense(*operands(), bias=dev(torch.zeros(300, dtype=BF16))),
    "grouped_without_offsets": lambda: ops.fp8_grouped(*operands(E=3), None),
    "grouped_of_one_matrix": lambda: ops.fp8_grouped(*operands(), OFFSETS),
    "grouped_offsets_size": lambda: ops.fp8_grouped(*operands(E=4), OFFSETS),
    "grouped_offsets_int64": lambda: ops.fp8_grouped(*operands(E=3), dev(OFFSETS.to(torch.int64))),
    "grouped_few_out_rows": lambda: ops.fp8_grouped(*operands(E=3), OFFSETS, out_rows=dev(torch.zeros(4, dtype=torch.int32))),
    "grouped_few_row_scales": lambda: ops.fp8_grouped(*operands(E=3), OFFSETS, row_scale=dev(torch.zeros(4))),
    "grouped_scale_rows_alone": lambda: ops.fp8_grouped(*operands(E=3), OFFSETS, scale_rows=dev(torch.zeros(5, dtype=torch.int32))),
    "grouped_experts_apart": lambda: ops.fp8_grouped(*operands(E=3)[:2], dev(ops.fp8_empty((6, 300, 200), "cpu")[::2]), operands(E=3)[3], OFFSETS),
    "swiglu_odd_rows": lambda: ops.fp8_swiglu(*operands(N=257)),
    "swiglu_offsets_for_one_matrix": lambda: ops.fp8_swiglu(*operands(N=256), OFFSETS),
    "swiglu_of_bf16_weights": lambda: ops.fp8_swiglu(*operands()[:2], dev(torch.zeros(256, 200, dtype=BF16)), dev(torch.ones(2, 2))),
}


@pytest.mark.parametrize("name", sorted(REFUSED))
def test_refused(calls, name):
    with pytest.raises(KernelError):
        REFUSED[name]()
    assert not calls


def few(T=3, E=6, H=64, I=32, k=2, w8=False, **more):
    """A call of moe_few with some of its arguments replaced."""
    args = {"h": dev(torch.zeros(T, H, dtype=BF16)), "router": dev(torch.zeros(E, H)),
            "gate_up": dev(ops.fp8_empty((E, 2 * I, H), "cpu") if w8 else torch.zeros(E, 2 * I, H, dtype=BF16)),
            "down": dev(ops.fp8_empty((E, H, I), "cpu") if w8 else torch.zeros(E, H, I, dtype=BF16))}
    if w8:
        args["gate_up_scale"] = dev(torch.ones(E, ops.fp8_blocks(2 * I), ops.fp8_blocks(H)))
        args["down_scale"] = dev(torch.ones(E, ops.fp8_blocks(H), ops.fp8_blocks(I)))
    args.update(more)
    return ops.moe_few(args.pop("h"), args.pop("router"), args.pop("gate_up"), args.pop("down"), k, **args)


def test_few_calls_that_are_taken(calls):
    few()
    few(w8=True, H=63, I=34)
    few(T=16, k=6, bias=dev(torch.zeros(6)), correction=dev(torch.zeros(6)), scoring="softmax_chosen", weights_on="input", out_dtype=BF16)
    assert [s for s, _ in calls] == ["sharpi_moe_few"] * 3


FEW_REFUSED = {
    "on_the_cpu": dict(h=torch.zeros(3, 64, dtype=BF16)),
    "float32_rows": dict(h=dev(torch.zeros(3, 64))),
    "17_tokens": dict(T=17),
    "no_experts_a_token": dict(k=0),
    "more_experts_a_token_than_there_are": dict(k=7),
    "33_experts_a_token": dict(E=40, k=33),
    "1025_experts": dict(E=1025, H=8, I=8),
    "router_shape": dict(router=dev(torch.zeros(5, 64))),
    "router_bf16": dict(router=dev(torch.zeros(6, 64, dtype=BF16))),
    "gate_up_shape": dict(gate_up=dev(torch.zeros(6, 63, 64, dtype=BF16))),
    "gate_up_float32": dict(gate_up=dev(torch.zeros(6, 64, 64))),
    "down_shape": dict(down=dev(torch.zeros(6, 32, 64, dtype=BF16))),
    "down_on_the_cpu": dict(down=torch.zeros(6, 64, 32, dtype=BF16)),
    "widths_of_bf16_weights": dict(H=60),
    "inner_width_of_bf16_weights": dict(I=28),
    "odd_inner_width": dict(w8=True, I=33),
    "one_scale_alone": dict(w8=True, down_scale=None),
    "scale_shape": dict(w8=True, down_scale=dev(torch.ones(6, 2, 1))),
    "8_bit_weights_without_scales": dict(w8=True, gate_up_scale=None, down_scale=None),
    "rows_off_16_bytes": dict(gate_up=dev(torch.zeros(6, 64, 68, dtype=BF16)[..., 4:])),
    "rows_apart_unevenly": dict(gate_up=dev(torch.zeros(6, 70, 64, dtype=BF16)[:, :64])),
    "unknown_scoring": dict(scoring="softmax"),
    "unknown_place_of_weights": dict(weights_on="both"),
    "bias_size": dict(bias=dev(torch.zeros(5))),
    "correction_dtype": dict(correction=dev(torch.zeros(6, dtype=BF16))),
    "h32_shape": dict(h32=dev(torch.zeros(2, 64))),
    "add_bf16": dict(add=dev(torch.zeros(3, 64, dtype=BF16))),
    "out_shape": dict(out=dev(torch.zeros(3, 65))),
    "out_float16": dict(out_dtype=torch.float16),
}


@pytest.mark.parametrize("name", sorted(FEW_REFUSED))
def test_few_refused(calls, name):
    with pytest.raises(KernelError):
        few(**FEW_REFUSED[name])
    assert not calls


def test_another_device_is_refused(calls, monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    for call in (lambda: ops.fp8_rows(dev(torch.zeros(5, 200))), lambda: ops.fp8_weight(dev(torch.zeros(5, 200))),
                 lambda: ops.fp8_dense(*operands()), lambda: ops.fp8_swiglu(*operands(N=256)), few):
        with pytest.raises(KernelError, match="current device"):
            call()
    assert not calls
