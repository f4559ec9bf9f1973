"""The oracle of the serving operators against cases worked out by hand, and the refusals of the
entry points: descriptors are checked before any CUDA call, so both run without a GPU."""
import ctypes

import numpy as np
import pytest

from compiler_b200 import kernels, ops
from compiler_b200.registry import UnsupportedLaunch, default_registry
from compiler_b200.runtime import abi
from oracle import oracle, serving


def test_nearest_rounds_ties_to_even_and_keeps_what_the_type_holds():
    assert serving.nearest(1.0 + 2.0 ** -8, "bfloat16") == 1.0                # tie: 1.0 is even
    assert serving.nearest(1.0 + 3 * 2.0 ** -8, "bfloat16") == 1.0 + 2.0 ** -6
    assert serving.nearest(1.0 + 2.0 ** -8 + 2.0 ** -40, "bfloat16") == 1.0 + 2.0 ** -7
    assert serving.nearest(2.0 ** -24 * 1.5, "float16") == 2.0 ** -23         # below the normal range
    rng = np.random.default_rng(0)
    x = rng.standard_normal(4096).astype(np.float32)
    assert np.array_equal(serving.nearest(x, "bfloat16"), oracle.bf16_round(x))
    assert np.array_equal(serving.nearest(x, "float16"), x.astype(np.float16))
    assert np.isnan(serving.nearest(np.nan, "float16")) and serving.nearest(np.inf, "bfloat16") == np.inf


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_keeps_lengths_and_turns_a_quarter(interleaved):
    x = np.arange(1.0, 13.0).reshape(1, 2, 6)
    cos, sin = np.zeros((1, 2), np.float32), np.ones((1, 2), np.float32)
    y = serving.rotate(x, cos, sin, interleaved)
    assert np.array_equal(y[..., 4:], x[..., 4:])                # behind the rotated part
    expected = [-2, 1, -4, 3] if interleaved else [-3, -4, 1, 2]
    assert np.array_equal(y[0, 0, :4], expected)
    angle = np.random.default_rng(1).uniform(0, 6, (1, 2))
    z = serving.rotate(x, np.cos(angle), np.sin(angle), interleaved)
    assert np.allclose((z ** 2).sum(-1), (x ** 2).sum(-1))


def test_four_bit_rows():
    codes, scale, low = serving.four_bits(np.array([[0.0, 15.0, 0.5, 1.5], [2.0, 2.0, 2.0, 2.0]]), "float16")
    assert codes.tolist() == [[0, 15, 0, 2], [0, 0, 0, 0]]        # ties to even; a constant row
    assert scale.tolist() == [1.0, 0.0] and low.tolist() == [0.0, 2.0]
    assert np.array_equal(serving.unpack(serving.pack(codes)), codes)
    assert serving.pack(codes)[0].tolist() == [0xf0, 0x20]
    rng = np.random.default_rng(2)
    rows = serving.nearest(rng.standard_normal((64, 128)), "bfloat16")
    codes, scale, low = serving.four_bits(rows, "bfloat16")
    # half a step, and what the rounding of the scale (2^-9 of 15 steps at most) takes off the end
    assert (np.abs(serving.stands_for(codes, scale, low) - rows) <= scale[:, None] * 0.54).all()


def test_attention_rows_against_the_dense_oracle():
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((5, 4, 16)), rng.standard_normal((5, 2, 16)), rng.standard_normal((5, 2, 16))
    out, lse, mass, top = serving.attention_rows(q, k, v, 0.25, True)
    dense, dense_lse = oracle.attention_ref(q.transpose(1, 0, 2)[None], np.repeat(k, 2, 1).transpose(1, 0, 2)[None],
                                            np.repeat(v, 2, 1).transpose(1, 0, 2)[None], 0.25, True)
    assert np.allclose(out, dense[0].transpose(1, 0, 2)) and np.allclose(lse, dense_lse[0].T)
    assert (mass >= np.abs(out) - 1e-12).all() and (top > 0).all()
    # more queries than keys: the first rows see nothing
    out, lse, _, _ = serving.attention_rows(q, k[:2], v[:2], 0.25, True)
    assert (out[:3] == 0).all() and np.isposinf(lse[:3]).all() and np.isfinite(lse[3:]).all()


def test_quantized_rows():
    codes, scale = serving.quantize_rows(np.array([[127.0, -127.0, 0.5, 1.5, -2.5], [0, 0, 0, 0, 0]]))
    assert codes.tolist() == [[127, -127, 0, 2, -2], [0, 0, 0, 0, 0]] and scale.tolist() == [1.0, 0.0]


# ------------------------------------------------------------------------------- refusals
class Fake:
    """A device array that is never looked at."""

    def __init__(self, shape, dtype, strides=None, ptr=0x10000):
        self.shape, self.dtype, self._strides, self._ptr = tuple(shape), dtype, strides, ptr

    def data_ptr(self):
        return self._ptr

    def stride(self):
        if self._strides is not None:
            return self._strides
        out, step = [], 1
        for extent in reversed(self.shape):
            out.append(step)
            step *= max(extent, 1)
        return tuple(reversed(out))


def _append_args(bits=16, dtype="bfloat16", t=3, hk=2, d=64, pages=4, block=16):
    row = d if bits == 16 else d // 2
    cache = "uint8" if bits == 4 else dtype
    args = {"k": Fake((t, hk, d), dtype), "v": Fake((t, hk, d), dtype),
            "k_cache": Fake((pages, hk, block, row), cache), "v_cache": Fake((pages, hk, block, row), cache),
            "page_table": Fake((2, 3), "int32"), "seq": Fake((t,), "int32"), "pos": Fake((t,), "int32")}
    if bits == 4:
        args.update(k_params=Fake((pages, hk, block, 2), dtype), v_params=Fake((pages, hk, block, 2), dtype))
    return args


APPEND_REFUSALS = [
    (16, {"v": Fake((3, 2, 32), "bfloat16")}, "k and v"),
    (16, {"v": Fake((3, 2, 64), "float16")}, "dtypes"),
    (16, {"k": Fake((3, 2, 64), "int8"), "v": Fake((3, 2, 64), "int8")}, "dtype"),
    (16, {"k": Fake((3, 2, 64), "bfloat16", (256, 128, 2))}, "unit last stride"),
    (16, {"k_cache": Fake((4, 2, 16, 64), "float16")}, "caches"),
    (16, {"k_cache": Fake((4, 2, 8, 64), "bfloat16")}, "both caches"),
    (16, {"k_cache": Fake((4, 2, 16, 64), "bfloat16", (4096, 2048, 1, 16))}, "unit last stride"),
    (16, {"v_cache": Fake((5, 2, 16, 64), "bfloat16")}, "both caches"),
    (16, {"k_params": Fake((4, 2, 16, 2), "bfloat16")}, "params"),
    (4, {"k_params": None}, "params"),
    (4, {"v_params": Fake((4, 2, 16, 2), "float32")}, "k's dtype"),
    (4, {"v_params": Fake((4, 2, 16, 1), "bfloat16")}, "params must be"),
    (4, {"k_cache": Fake((4, 2, 16, 64), "uint8")}, "both caches"),
    (16, {"page_table": Fake((2, 3), "int64")}, "int32"),
    (16, {"page_table": Fake((2, 3), "int32", (1, 2))}, "page_table"),
    (16, {"seq": Fake((4,), "int32")}, "one entry per token"),
    (16, {"pos": Fake((3,), "int32", (2,))}, "contiguous"),
    (16, {"cos": Fake((9, 32), "float32")}, "come together"),
    (16, {"cos": Fake((9, 33), "float32"), "sin": Fake((9, 33), "float32")}, "rotated elements"),
    (16, {"cos": Fake((9, 32), "bfloat16"), "sin": Fake((9, 32), "bfloat16")}, "f32"),
    (16, {"cos": Fake((9, 32), "float32"), "sin": Fake((8, 32), "float32")}, "differ"),
    (16, {"q": Fake((3, 4, 64), "bfloat16")}, "come together"),
    (16, {"q": Fake((3, 4, 64), "bfloat16"), "q_out": Fake((3, 5, 64), "bfloat16")}, "q and q_out"),
    (16, {"k_out": Fake((3, 2, 64), "float32")}, "k_out"),
    (16, {"k": Fake((3, 2, 64), "bfloat16", ptr=0)}, "null data"),
]


@pytest.mark.parametrize("bits, change, text", APPEND_REFUSALS)
def test_append_refusals(bits, change, text):
    args = {**_append_args(bits), **change}
    with pytest.raises(abi.B200Error) as err:
        ops.kv_append(**args)
    assert err.value.status == abi.REJECTED and text in err.value.detail


def test_append_of_nothing_and_odd_four_bit_heads():
    empty = _append_args(t=0)
    ops.kv_append(**empty)  # no device needed
    odd = _append_args(bits=4, d=64)
    odd["k"] = odd["v"] = Fake((3, 2, 63), "bfloat16")
    with pytest.raises(abi.B200Error):
        ops.kv_append(**odd)


def _attend_args(bits=16, dtype="float16", t=4, h=4, hk=2, d=64, z=2, pages=4, block=16):
    row = d if bits == 16 else d // 2
    cache = "uint8" if bits == 4 else dtype
    args = {"q": Fake((t, h, d), dtype), "k_cache": Fake((pages, hk, block, row), cache),
            "v_cache": Fake((pages, hk, block, row), cache), "page_table": Fake((z, 3), "int32"),
            "lengths": Fake((z,), "int32"), "out": Fake((t, h, d), dtype),
            "workspace": Fake((ops.attention_paged_workspace(t, h, hk, d),), "uint8")}
    if bits == 4:
        args.update(k_params=Fake((pages, hk, block, 2), dtype), v_params=Fake((pages, hk, block, 2), dtype))
    return args


ATTEND_REFUSALS = [
    (16, {"q": Fake((4, 3, 64), "float16"), "out": Fake((4, 3, 64), "float16")}, "multiple"),
    (16, {"out": Fake((4, 4, 32), "float16")}, "out must be"),
    (16, {"out": Fake((4, 4, 64), "float32")}, "out must be"),
    (16, {"q": Fake((4, 4, 64), "float16", (512, 1, 8))}, "unit last stride"),
    (16, {"k_cache": Fake((4, 2, 16, 64), "bfloat16")}, "caches"),
    (16, {"v_cache": Fake((4, 2, 16, 32), "float16")}, "both caches"),
    (4, {"k_params": None}, "params"),
    (4, {"k_params": Fake((4, 2, 16, 2), "bfloat16")}, "q's dtype"),
    (16, {"lengths": Fake((3,), "int32")}, "lengths"),
    (16, {"lengths": Fake((2,), "int64")}, "int32"),
    (16, {"page_table": Fake((2, 3), "float32")}, "int32"),
    (16, {"cu_seqlens_q": Fake((2,), "int32")}, "cu_seqlens_q"),
    (16, {"q": Fake((5, 4, 64), "float16"), "out": Fake((5, 4, 64), "float16")}, "divide"),
    (16, {"lse": Fake((4, 4), "float16")}, "lse"),
    (16, {"scale": -1.0}, "scale"),
    (16, {"scale": float("nan")}, "scale"),
    (16, {"scale": float("inf")}, "scale"),
    (16, {"workspace": Fake((16,), "uint8")}, "workspace"),
    (16, {"workspace": Fake((1 << 26,), "uint8", ptr=0x10008)}, "workspace"),
]


@pytest.mark.parametrize("bits, change, text", ATTEND_REFUSALS)
def test_attention_refusals(bits, change, text):
    with pytest.raises(abi.B200Error) as err:
        ops.attention_paged(**{**_attend_args(bits), **change})
    assert err.value.status == abi.REJECTED and text in err.value.detail


def test_workspace_query():
    assert ops.attention_paged_workspace(1, 8, 8, 64) > 0
    for bad in ((1, 3, 2, 64), (1, 2, 2, 0), (1, 2, 2, 513), (-1, 2, 2, 64)):
        with pytest.raises(abi.B200Error):
            ops.attention_paged_workspace(*bad)
    assert abi.lib().b200_attn_paged_workspace(1, 2, 2, 64, None) == abi.USAGE


LINEAR_REFUSALS = [
    ({"x": Fake((4, 32), "uint8")}, abi.REJECTED, "int8"),
    ({"w": Fake((8, 31), "int8")}, abi.REJECTED, "columns"),
    ({"x_scale": Fake((5,), "float32")}, abi.REJECTED, "x_scale"),
    ({"w_scale": Fake((8,), "float16")}, abi.REJECTED, "w_scale"),
    ({"y": Fake((4, 9), "float16")}, abi.REJECTED, "y must"),
    ({"y": Fake((4, 8), "int8")}, abi.REJECTED, "y must"),
    ({"x": Fake((4, 32), "int8", (64, 2))}, abi.REJECTED, "unit column"),
    ({"bias": Fake((7,), "float32")}, abi.REJECTED, "bias"),
    ({"act": abi.ACT_SWIGLU}, abi.USAGE, "activation"),
    ({"act": 77}, abi.USAGE, "activation"),
    ({"x": Fake((4, 1 << 18), "int8"), "w": Fake((8, 1 << 18), "int8")}, abi.REJECTED, "K "),
]


@pytest.mark.parametrize("change, status, text", LINEAR_REFUSALS)
def test_linear_int8_refusals(change, status, text):
    args = {"x": Fake((4, 32), "int8"), "x_scale": Fake((4,), "float32"), "w": Fake((8, 32), "int8"),
            "w_scale": Fake((8,), "float32"), "y": Fake((4, 8), "float16"), **change}
    with pytest.raises(abi.B200Error) as err:
        ops.linear_int8(**args)
    assert err.value.status == status and text in err.value.detail


def test_quantize_refusals():
    for x, out, scale in ((Fake((4, 8), "int8"), Fake((4, 8), "int8"), Fake((4,), "float32")),
                          (Fake((4, 8), "float16"), Fake((4, 8), "uint8"), Fake((4,), "float32")),
                          (Fake((4, 8), "float16"), Fake((4, 7), "int8"), Fake((4,), "float32")),
                          (Fake((4, 8), "float16"), Fake((4, 8), "int8"), Fake((4,), "float16")),
                          (Fake((4, 8), "float16", (16, 2)), Fake((4, 8), "int8"), Fake((4,), "float32"))):
        with pytest.raises(abi.B200Error):
            ops.quantize_rows(x, out, scale)
    ops.quantize_rows(Fake((0, 8), "float16"), Fake((0, 8), "int8"), Fake((0,), "float32"))


def test_null_descriptors_are_usage_errors():
    lib = abi.lib()
    assert lib.b200_kv_append(*[None] * 11, 0, *[None] * 4, None) == abi.USAGE
    assert lib.b200_attn_paged(*[None] * 10, 1.0, 1, None, 0, None) == abi.USAGE
    assert lib.b200_linear_int8(*[None] * 6, 0, None) == abi.USAGE
    assert lib.b200_quantize_rows(None, None, None, None) == abi.USAGE


def test_handles_resolve_and_check_the_cache_format():
    registry = default_registry()
    for handle in (kernels.kv_append_kernel, kernels.paged_attention_kernel, kernels.quantize_rows_kernel,
                   kernels.linear_int8_kernel):
        assert registry.supports(handle) and not registry.reads_device(handle)
    values = dict(k_ptr=None, v_ptr=None, k_cache_ptr=Fake((64,), "uint8"), v_cache_ptr=Fake((64,), "uint8"),
                  k_params_ptr=None, v_params_ptr=None, page_table_ptr=Fake((2,), "int32"), seq_ptr=None,
                  pos_ptr=None, cos_ptr=None, sin_ptr=None, q_ptr=None, q_out_ptr=None, T=1, Z=1, WIDTH=1, H=1,
                  H_KV=1, HEAD_DIM=64, ROT_DIM=0, PAGES=1, BLOCK=1, ANGLES=0, BITS=16, INTERLEAVED=False)
    with pytest.raises(UnsupportedLaunch) as err:
        registry.launch(None, kernels.kv_append_kernel, (1,), list(values.values()), {})
    assert err.value.construct == "BITS"
