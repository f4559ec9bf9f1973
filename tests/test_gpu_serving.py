"""Serving operators on the GPU: paged append with rotation, attention over 16- and 4-bit pages, int8
linear layers, against the float64 oracle.

Tolerances are derived, not tuned.  The append is exact by its definition (one rounding of the
rotated value; codes decided by the 64-bit quotient), and so are the int8 codes.  Attention: the
scores are 32-bit sums of D products of which each adds at most 2^-23 of the running magnitude, a
relative error of (D + 16) 2^-23 of `top` = scale * sum |q k| (4-bit rows: of |low| + 15 scale in the
place of |k|); an error e of the scores moves every weight by 2e at most.  Weights may be rounded to
the query's 16-bit type once, 2^-9 (bf16) or 2^-11 (fp16), and the result is rounded once.  All of
this is counted against `mass` = sum p |v| (4-bit: p (|low| + 15 scale)).
"""
import zlib

import numpy as np
import pytest

from compiler_b200 import graph, harness, kernels, ops
from compiler_b200.registry import _View
from compiler_b200.runtime import abi
from oracle import oracle, serving

pytestmark = pytest.mark.gpu


def _rng(*parts):
    return np.random.default_rng(zlib.crc32(repr(parts).encode()))


def _up(device, values, dtype):
    """float64 values that `dtype` holds -> device."""
    values = np.asarray(values)
    if dtype in ("bfloat16", "float32"):
        return device.upload(values.astype(np.float32), dtype)
    return device.upload(values.astype(dtype), dtype)


def _down(device, buffer):
    return np.asarray(device.download(buffer), dtype=np.float64)


class Paged:
    """One side of a paged cache: contiguous device memory, viewed as [pages, heads, block, ...]."""

    def __init__(self, device, values, dtype, order):
        self.device, self.order = device, order
        self.shape = values.shape
        host = values if order == "head" else values.transpose(0, 2, 1, 3)
        self.buffer = (device.upload(np.ascontiguousarray(host), "uint8") if dtype == "uint8"
                       else _up(device, host, dtype))
        p, h, b, d = values.shape
        strides = (h * b * d, b * d, d, 1) if order == "head" else (b * h * d, d, h * d, 1)
        self.view = _View(self.buffer, values.shape, strides)

    def read(self):
        host = self.device.download(self.buffer)
        p, h, b, d = self.shape
        if self.order == "token":
            host = host.reshape(p, b, h, d).transpose(0, 2, 1, 3)
        return np.asarray(host if host.dtype == np.uint8 else host.astype(np.float64)).reshape(self.shape)


def _angles(positions, half):
    angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(half) / max(half, 1))
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


# ---------------------------------------------------------------------------------- append
APPEND = [
    # dtype, bits, D, R, interleaved, H, H_KV, block, order
    ("bfloat16", 16, 128, 128, False, 8, 2, 16, "head"),
    ("float16", 16, 128, 64, True, 4, 4, 32, "token"),
    ("float32", 32, 64, 64, False, 2, 1, 5, "head"),
    ("bfloat16", 16, 40, 24, False, 3, 3, 7, "token"),
    ("float16", 16, 33, 6, True, 1, 1, 1, "head"),
    ("bfloat16", 16, 256, 0, False, 0, 2, 16, "head"),
    ("float16", 16, 512, 512, True, 2, 1, 16, "head"),
    ("bfloat16", 4, 128, 128, False, 8, 2, 16, "head"),
    ("float16", 4, 128, 128, True, 4, 2, 48, "token"),
    ("bfloat16", 4, 64, 32, False, 5, 1, 64, "head"),
    ("float16", 4, 64, 64, False, 0, 8, 16, "token"),
    ("float32", 4, 64, 16, False, 2, 2, 16, "head"),
    ("bfloat16", 4, 48, 48, False, 2, 1, 3, "head"),
    ("float16", 4, 10, 4, True, 1, 1, 16, "head"),
    ("float16", 4, 256, 256, False, 2, 1, 16, "token"),
]


@pytest.mark.parametrize("tokens", [1, 37, 300])
@pytest.mark.parametrize("dtype, bits, dim, rot, interleaved, heads, kv, block, order", APPEND)
def test_append(device, dtype, bits, dim, rot, interleaved, heads, kv, block, order, tokens):
    rng = _rng(dtype, bits, dim, rot, interleaved, kv, block, tokens)
    seqs = min(3, tokens)
    # ragged spans with an offset each, and padding tokens between them
    spans = [int(n) for n in np.diff([0, *sorted(rng.integers(0, tokens + 1, seqs - 1)), tokens])]
    starts = rng.integers(0, 50, seqs)
    seq = np.repeat(np.arange(seqs), spans).astype(np.int32)
    pos = np.concatenate([starts[z] + np.arange(n) for z, n in enumerate(spans)]).astype(np.int32)
    seq[rng.random(tokens) < 0.1] = -1
    width = int(max(starts + spans)) // block + 1
    pages = seqs * width + 2
    table = rng.permutation(pages)[:seqs * width].reshape(seqs, width).astype(np.int32)
    # q, k, v as slices of one projection, as a layer hands them over
    fused = serving.nearest(rng.standard_normal((tokens, heads + 2 * kv, dim)) * 2, dtype)
    fused[..., ::7] += serving.nearest(np.float64(1.0), dtype) * 3
    fused = serving.nearest(fused, dtype)
    q, k, v = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
    base = _up(device, fused, dtype)
    row = (heads + 2 * kv) * dim

    def part(first, count):
        return _View(base, (tokens, count, dim), (row, dim, 1), offset=first * dim)

    shape = (pages, kv, block, dim if bits != 4 else dim // 2)
    if bits == 4:
        before = [rng.integers(0, 256, shape).astype(np.uint8) for _ in range(2)]
        par_before = [serving.nearest(rng.standard_normal((pages, kv, block, 2)), dtype) for _ in range(2)]
        caches = [Paged(device, c, "uint8", order) for c in before]
        params = [Paged(device, c, dtype, order) for c in par_before]
    else:
        before = [serving.nearest(rng.standard_normal(shape), dtype) for _ in range(2)]
        caches, params = [Paged(device, c, dtype, order) for c in before], None
    cos, sin = _angles(int(pos.max()) + 1, rot // 2)
    extra = {}
    if rot:
        extra.update(cos=device.upload(cos), sin=device.upload(sin), interleaved=interleaved)
    if heads:
        q_out = device.upload(np.full((tokens, heads, dim), 7, np.float32 if dtype != "float16" else np.float16), dtype)
        extra.update(q=part(0, heads), q_out=q_out)
    if params:
        extra.update(k_params=params[0].view, v_params=params[1].view)
    with_copies = tokens != 37
    if with_copies:
        k_out, v_out = (device.alloc((tokens, kv, dim), dtype) for _ in range(2))
        extra.update(k_out=k_out, v_out=v_out)
    ops.kv_append(part(heads, kv), part(heads + kv, kv), caches[0].view, caches[1].view,
                  device.upload(table), device.upload(seq), device.upload(pos), **extra)
    device.check_status()

    live = seq >= 0
    turn = lambda x: serving.nearest(serving.rotate(x, cos[pos], sin[pos], interleaved), dtype)  # noqa: E731
    if heads:
        got = _down(device, q_out)
        assert np.array_equal(got[live], turn(q)[live])
        assert (got[~live] == 7).all()
    for side, rows, cache, old in ((0, turn(k), caches[0], before[0]), (1, v, caches[1], before[1])):
        expected = old.copy()
        where = (table[seq[live], pos[live] // block], slice(None), pos[live] % block)
        if bits == 4:
            codes, scale, low = serving.four_bits(rows, dtype)
            expected[where] = serving.pack(codes)[live]
            par = par_before[side].copy()
            par[where] = np.stack((scale, low), -1)[live]
            assert np.array_equal(params[side].read(), par)
            rows = serving.stands_for(codes, scale, low)
        else:
            expected[where] = rows[live]
        assert np.array_equal(cache.read(), expected)
        if with_copies:
            got = _down(device, (k_out, v_out)[side])[live]
            # a code's value is rounded to 32 bits and then to the row's type
            bound = np.abs(rows[live]) * (serving.half_step(dtype) + 2.0 ** -23) + 2.0 ** -24
            assert (np.abs(got - rows[live]) <= (bound if bits == 4 else 0)).all()


@pytest.mark.parametrize("dtype, bits, dim", [("bfloat16", 16, 128), ("float16", 16, 36), ("float16", 4, 128)])
def test_append_in_place_and_at_far_positions(device, dtype, bits, dim):
    """q_out = q and k_out = k; positions beyond 2^17, where a page lies far behind the base."""
    rng = _rng(dtype, dim)
    tokens, far = 5, 140001
    x = {n: serving.nearest(rng.standard_normal((tokens, h, dim)), dtype) for n, h in (("q", 4), ("k", 2), ("v", 2))}
    d = {n: _up(device, t, dtype) for n, t in x.items()}
    block = 16
    table = np.full((1, (far + tokens) // block + 1), -1, np.int32)
    table[0, far // block:] = np.arange(table.shape[1] - far // block)
    pages = int(table.max()) + 1
    cos, sin = _angles(far + tokens, dim // 2)
    row = dim if bits == 16 else dim // 2
    zero = np.zeros((pages, 2, block, row), np.uint8 if bits == 4 else np.float64)
    caches = [Paged(device, zero, "uint8" if bits == 4 else dtype, "head") for _ in range(2)]
    extra = {}
    if bits == 4:
        params = [Paged(device, np.zeros((pages, 2, block, 2)), dtype, "head") for _ in range(2)]
        extra = {"k_params": params[0].view, "v_params": params[1].view}
    pos = (far + np.arange(tokens)).astype(np.int32)
    ops.kv_append(d["k"], d["v"], caches[0].view, caches[1].view, device.upload(table),
                  device.upload(np.zeros(tokens, np.int32)), device.upload(pos), cos=device.upload(cos),
                  sin=device.upload(sin), q=d["q"], q_out=d["q"], k_out=d["k"], v_out=d["v"], **extra)
    device.check_status()
    q, k = (serving.nearest(serving.rotate(x[n], cos[pos], sin[pos]), dtype) for n in ("q", "k"))
    assert np.array_equal(_down(device, d["q"]), q)
    held = caches[0].read()[table[0, pos // block], :, pos % block]
    if bits == 16:
        assert np.array_equal(held, k) and np.array_equal(_down(device, d["k"]), k)
    else:
        assert np.array_equal(held, serving.pack(serving.four_bits(k, dtype)[0]))


@pytest.mark.parametrize("dim", [64, 20])
def test_append_leaves_out_what_has_no_place(device, dim):
    """Sequences, positions and pages outside their tables: reported, left out whole."""
    tokens, block = 6, 16
    seq = np.array([0, 5, 0, 0, 1, 0], np.int32)
    pos = np.array([0, 0, 99, -3, 0, 17], np.int32)      # 99: behind the table's two pages
    table = np.array([[2, 0], [77, -1]], np.int32)       # sequence 1 names a page that is not there
    rng = _rng("bad", dim)
    x = serving.nearest(rng.standard_normal((tokens, 1, dim)), "bfloat16")
    dx = _up(device, x, "bfloat16")
    caches = [Paged(device, np.zeros((3, 1, block, dim)), "bfloat16", "head") for _ in range(2)]
    q_out = _up(device, np.full((tokens, 1, dim), 7.0), "bfloat16")
    ops.kv_append(dx, dx, caches[0].view, caches[1].view, device.upload(table), device.upload(seq),
                  device.upload(pos), q=dx, q_out=q_out)
    with pytest.raises(abi.B200Error) as err:
        device.check_status()
    assert err.value.status == abi.REJECTED
    device.check_status()  # read and cleared
    expected = np.zeros((3, 1, block, dim))
    expected[2, 0, 0], expected[0, 0, 1] = x[0, 0], x[5, 0]
    assert np.array_equal(caches[0].read(), expected) and np.array_equal(caches[1].read(), expected)
    got = _down(device, q_out)
    assert np.array_equal(got[[0, 5]], x[[0, 5]]) and (got[1:5] == 7).all()
    # a position behind the table of angles
    cos, sin = _angles(4, dim // 2)
    ops.kv_append(dx, dx, caches[0].view, caches[1].view, device.upload(table),
                  device.upload(np.zeros(tokens, np.int32)),
                  device.upload(np.arange(tokens, dtype=np.int32)), cos=device.upload(cos), sin=device.upload(sin))
    with pytest.raises(abi.B200Error):
        device.check_status()
    assert (caches[1].read()[2, 0, 4:] == 0).all() and np.array_equal(caches[1].read()[2, 0, 3], x[3, 0])


@pytest.mark.parametrize("dim", [128, 12])
def test_append_rows_without_a_range(device, dim):
    """Constant rows, tiny ranges, infinities and NaN in a 4-bit cache."""
    rows = np.zeros((6, 1, dim))
    rows[1] = 3.0
    rows[2, 0, ::2] = 2.0 ** -24          # the scale rounds to zero
    rows[3, 0, 1] = np.inf
    rows[4, 0, 2] = np.nan
    rows[5, 0, ::3] = -60000.0
    rows[5, 0, 1] = 60000.0
    d = _up(device, rows, "float16")
    caches = [Paged(device, np.zeros((1, 1, 16, dim // 2), np.uint8), "uint8", "head") for _ in range(2)]
    params = [Paged(device, np.zeros((1, 1, 16, 2)), "float16", "head") for _ in range(2)]
    out = device.alloc(rows.shape, "float16")
    ops.kv_append(d, d, caches[0].view, caches[1].view, device.upload(np.zeros((1, 1), np.int32)),
                  device.upload(np.zeros(6, np.int32)), device.upload(np.arange(6, dtype=np.int32)),
                  k_params=params[0].view, v_params=params[1].view, k_out=out)
    device.check_status()
    got = _down(device, out)[:, 0]
    assert (got[0] == 0).all() and (got[1] == 3).all() and (got[2] == 0).all()
    assert np.isnan(got[3]).all() and np.isnan(got[4]).all()
    codes, scale, low = serving.four_bits(rows[5], "float16")
    assert np.array_equal(caches[0].read()[0, 0, 5], serving.pack(codes)[0])
    assert np.array_equal(params[0].read()[0, 0, 5], [scale[0], low[0]])


# ------------------------------------------------------------------------------- attention
def _make_cache(device, rng, dtype, bits, lengths, kv, dim, block, order, garbage=True, room=0):
    """Pages in a random order; rows behind the last key hold NaN, infinities or large codes.  The
    page table has room for ``room`` keys at least (how long contexts may get decides the kernel)."""
    counts = [-(-n // block) for n in lengths]
    width = max(max(counts + [1]) + 1, -(-room // block))
    pages = sum(counts) + 1
    table = np.full((len(lengths), width), -1, np.int32)
    order_of = rng.permutation(pages)
    at = 0
    for z, n in enumerate(counts):
        table[z, :n] = order_of[at:at + n]
        at += n
    sides = []
    for shift in (1.0, 0.3):
        rows = rng.standard_normal((pages, kv, block, dim)) + shift * rng.standard_normal((1, kv, 1, dim))
        rows = serving.nearest(rows, dtype)
        dead = np.ones((pages, block), bool)
        for z, n in enumerate(lengths):
            j = np.arange(n)
            dead[table[z, j // block], j % block] = False
        if bits == 4:
            codes, scale, low = serving.four_bits(rows, dtype)
            held = serving.stands_for(codes, scale, low)
            size = np.abs(low) + 15 * scale
            par = np.stack((scale, low), -1)
            if garbage:
                par.transpose(0, 2, 1, 3)[dead] = [np.nan, np.inf]
            sides.append((Paged(device, serving.pack(codes), "uint8", order), Paged(device, par, dtype, order),
                          held, np.broadcast_to(size[..., None], held.shape)))
        else:
            stored = rows.copy()
            if garbage:
                stored.transpose(0, 2, 1, 3)[dead] = np.nan
                stored.transpose(0, 2, 1, 3)[dead, :, ::2] = np.inf
            sides.append((Paged(device, stored, dtype, order), None, rows, np.abs(rows)))
    return table, sides


def _check_attention(device, dtype, q, out, lse, table, sides, lengths, spans, scale, causal, block):
    got, got_lse = _down(device, out), _down(device, lse)
    weight = {"bfloat16": 2.0 ** -9, "float16": 2.0 ** -11, "float32": 0.0}[dtype]
    dim = q.shape[-1]
    touched = np.zeros(q.shape[0], bool)
    for z, (begin, end) in enumerate(spans):
        k, v = (serving.gather(side[2], table[z], lengths[z], block) for side in sides)
        k_size, v_size = (serving.gather(side[3], table[z], lengths[z], block) for side in sides)
        touched[begin:end] = True
        if begin == end:
            continue
        ref, ref_lse, _, _ = serving.attention_rows(q[begin:end], k, v, scale, causal)
        # the magnitudes, by the same weights: sum p |v|, and the largest scale * sum |q| |k|
        top = np.zeros(ref_lse.shape)
        group = q.shape[1] // k.shape[1]
        if len(k):
            top = scale * np.einsum("nhd,jhd->njh", np.abs(q[begin:end]), np.repeat(k_size, group, 1)).max(1)
        mass = np.zeros(ref.shape)
        for i in range(end - begin):
            seen = max(0, min(lengths[z], lengths[z] - (end - begin) + i + 1)) if causal else lengths[z]
            for h in range(q.shape[1]):
                if seen:
                    s = scale * (k[:seen, h // group] @ q[begin + i, h])
                    p = np.exp(s - ref_lse[i, h])
                    mass[i, h] = p @ v_size[:seen, h // group]
        error = (dim + 16) * 2.0 ** -23 * top
        bound = mass * (weight + 2 * error + 16 * 2.0 ** -23 + len(k) * 2.0 ** -24)[..., None]
        bound = bound + np.abs(ref) * serving.half_step(dtype) * 1.01 + 2.0 ** -24
        bad = ~(np.abs(got[begin:end] - ref) <= bound)
        assert not bad.any(), (z, np.argwhere(bad)[:4], got[begin:end][bad][:4], ref[bad][:4], bound[bad][:4])
        empty = np.isposinf(ref_lse)
        assert np.array_equal(np.isposinf(got_lse[begin:end]), empty)
        assert (got[begin:end][empty] == 0).all()
        slack = error + 2.0 ** -21 * (1 + np.abs(np.where(empty, 0, ref_lse))) + len(k) * 2.0 ** -24
        assert (np.abs(got_lse[begin:end][~empty] - ref_lse[~empty]) <= slack[~empty]).all()
    assert (got[~touched] == 7).all() and (got_lse[~touched] == 7).all()


def _run_attention(device, dtype, bits, dim, heads, kv, block, order, lengths, counts, causal=True, scale=None,
                   extra_rows=0, stream=0, use_cu=True, garbage=True, spread=1.0, room=0):
    rng = _rng(dtype, bits, dim, heads, kv, block, order, tuple(lengths), tuple(counts), causal)
    table, sides = _make_cache(device, rng, dtype, bits, lengths, kv, dim, block, order, garbage, room)
    edges = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    tokens = int(edges[-1]) + extra_rows
    q = serving.nearest(rng.standard_normal((tokens, heads, dim)) * spread, dtype)
    # q and out as slices of wider rows
    wide = np.zeros((tokens, heads + 1, dim))
    wide[:, :heads] = q
    dq = _View(_up(device, wide, dtype), (tokens, heads, dim), ((heads + 1) * dim, dim, 1))
    out = _up(device, np.full((tokens, heads, dim), 7.0), dtype)
    lse = _up(device, np.full((tokens, heads), 7.0), "float32")
    scale = scale or dim ** -0.5
    work = device.alloc((ops.attention_paged_workspace(tokens, heads, kv, dim),), "uint8")
    ops.attention_paged(dq, sides[0][0].view, sides[1][0].view, device.upload(table),
                        device.upload(np.array(lengths, np.int32)), out, work,
                        k_params=sides[0][1].view if bits == 4 else None,
                        v_params=sides[1][1].view if bits == 4 else None,
                        cu_seqlens_q=device.upload(edges) if use_cu else None, lse=lse, scale=scale,
                        causal=causal, stream=stream)
    if stream:
        abi.check(abi.lib().b200_stream_sync(stream))
    device.check_status()
    spans = list(zip(edges[:-1].tolist(), edges[1:].tolist()))
    _check_attention(device, dtype, q, out, lse, table, sides, lengths, spans, scale, causal, block)


ATTEND = [
    # dtype, bits, D, H, H_KV, block, order
    ("bfloat16", 16, 128, 8, 2, 16, "head"),
    ("float16", 16, 128, 4, 4, 32, "token"),
    ("float16", 16, 64, 7, 1, 48, "token"),
    ("bfloat16", 16, 64, 16, 1, 128, "head"),
    ("bfloat16", 4, 128, 8, 2, 16, "head"),
    ("float16", 4, 128, 10, 2, 32, "token"),
    ("float16", 4, 64, 7, 1, 48, "head"),
    ("bfloat16", 4, 64, 24, 2, 64, "token"),
    ("bfloat16", 16, 128, 4, 2, 10, "head"),     # pages that are no multiple of a tile
    ("float16", 4, 128, 4, 2, 3, "token"),
    ("float32", 32, 64, 4, 2, 16, "head"),
    ("float32", 4, 128, 2, 1, 16, "head"),
    ("bfloat16", 16, 80, 4, 2, 16, "head"),
    ("float16", 4, 96, 4, 1, 16, "token"),
    ("float16", 16, 33, 2, 1, 7, "head"),
    ("bfloat16", 16, 256, 2, 1, 16, "head"),
]


@pytest.mark.parametrize("lengths, counts", [
    ([1], [1]),
    ([17, 1, 64, 255], [1, 1, 1, 1]),
    ([300, 0, 33, 16, 1], [3, 1, 0, 2, 4]),     # no keys; no queries; more queries than keys
    ([513, 130], [9, 37]),
])
@pytest.mark.parametrize("room", [0, 9000, 40000])
@pytest.mark.parametrize("dtype, bits, dim, heads, kv, block, order", ATTEND)
def test_attention(device, dtype, bits, dim, heads, kv, block, order, lengths, counts, room):
    _run_attention(device, dtype, bits, dim, heads, kv, block, order, lengths, counts, extra_rows=2, room=room)


@pytest.mark.parametrize("dtype, bits, dim", [("bfloat16", 16, 128), ("float16", 4, 128), ("float16", 4, 64),
                                              ("bfloat16", 4, 40)])
def test_attention_without_the_causal_mask(device, dtype, bits, dim):
    for room in (0, 9000, 40000):
        _run_attention(device, dtype, bits, dim, 4, 2, 16, "head", [100, 7, 31], [5, 5, 5], causal=False,
                       use_cu=False, room=room)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_attention_over_long_and_many(device, dtype, bits):
    """Rows cut between many CTAs, and more sequences than CTAs."""
    _run_attention(device, dtype, bits, 128, 4, 1, 64, "head", [9001], [1])
    rng = _rng("many", bits)
    lengths = [int(n) for n in rng.integers(0, 90, 700)]
    _run_attention(device, dtype, bits, 64, 2, 2, 16, "token", lengths, [1] * 700, use_cu=False)
    _run_attention(device, dtype, bits, 128, 8, 1, 32, "head", [int(n) for n in rng.integers(1, 700, 40)],
                   [int(n) for n in rng.integers(0, 6, 40)])


@pytest.mark.parametrize("heads, tokens", [(4, 1), (16, 1), (16, 2)])
@pytest.mark.parametrize("dtype, bits, dim", [("bfloat16", 16, 128), ("float16", 4, 128), ("bfloat16", 4, 64)])
def test_attention_of_an_item_in_very_many_pieces(device, dtype, bits, dim, heads, tokens):
    """More pieces than the join's shared memory takes at once."""
    _run_attention(device, dtype, bits, dim, heads, 1, 64, "head", [41003], [tokens], garbage=False)
    _run_attention(device, dtype, bits, dim, heads, 2, 64, "token", [20001, 5, 33001], [tokens, 1, 0], garbage=False,
                   room=50000)


@pytest.mark.parametrize("dtype, bits, dim", [("bfloat16", 16, 128), ("float16", 4, 128), ("bfloat16", 4, 64)])
def test_attention_of_a_prompt_behind_a_cached_part(device, dtype, bits, dim):
    """Hundreds of query tokens: many tiles of rows, each with a different last key."""
    _run_attention(device, dtype, bits, dim, 4, 1, 16, "head", [150, 70, 33], [120, 1, 33], room=0)
    _run_attention(device, dtype, bits, dim, 4, 1, 16, "head", [150, 70, 33], [120, 1, 33], room=9000)
    _run_attention(device, dtype, bits, dim, 4, 1, 16, "head", [150, 70, 33], [120, 1, 33], room=40000)


@pytest.mark.parametrize("bits", [16, 4])
def test_attention_peaked_and_flat_scores(device, bits):
    """Weights on one key, and scores whose running maximum keeps growing."""
    for room in (0, 9000, 40000):
        _run_attention(device, "bfloat16", bits, 128, 4, 1, 16, "head", [700], [1], spread=30.0, room=room)
        _run_attention(device, "float16", bits, 64, 4, 1, 16, "head", [700], [2], spread=1e-3, room=room)


@pytest.mark.parametrize("room", [0, 9000, 40000])
@pytest.mark.parametrize("dtype, bits, dim", [("bfloat16", 16, 128), ("bfloat16", 4, 128), ("float16", 16, 48)])
def test_attention_leaves_out_bad_pages_and_cuts_lengths(device, dtype, bits, dim, room):
    rng = _rng("pages", dtype, bits, dim)
    block, lengths = 16, [64, 50]
    table, sides = _make_cache(device, rng, dtype, bits, lengths, 1, dim, block, "head", room=room)
    q = serving.nearest(rng.standard_normal((2, 2, dim)), dtype)
    dq, work = _up(device, q, dtype), device.alloc((ops.attention_paged_workspace(2, 2, 1, dim),), "uint8")
    out, lse = device.alloc(q.shape, dtype), device.alloc((2, 2), "float32")
    params = dict(k_params=sides[0][1].view, v_params=sides[1][1].view) if bits == 4 else {}

    def run(table, lengths):
        ops.attention_paged(dq, sides[0][0].view, sides[1][0].view, device.upload(table),
                            device.upload(np.array(lengths, np.int32)), out, work, lse=lse, **params)

    broken = table.copy()
    broken[0, 1], broken[0, 3] = 1 << 20, -5
    run(broken, lengths)
    with pytest.raises(abi.B200Error) as err:
        device.check_status()
    assert err.value.status == abi.REJECTED
    keep = np.r_[0:16, 32:48]
    k, v = (serving.gather(side[2], table[0], 64, block)[keep] for side in sides)
    ref, ref_lse, _, _ = serving.attention_rows(q[:1], k, v, dim ** -0.5, False)
    assert np.abs(_down(device, out)[0] - ref[0]).max() <= 0.02 * np.abs(v).max()
    assert np.abs(_down(device, lse)[0] - ref_lse[0]).max() <= 1e-3
    # lengths outside the table: cut to it (pages that are there), negative ones to none
    narrow = np.ascontiguousarray(table[:, :3])
    run(narrow, [10 ** 6, -4])
    with pytest.raises(abi.B200Error):
        device.check_status()
    k, v = (serving.gather(side[2], table[0], 48, block) for side in sides)
    ref, ref_lse, _, _ = serving.attention_rows(q[:1], k, v, dim ** -0.5, False)
    assert np.abs(_down(device, lse)[0] - ref_lse[0]).max() <= 1e-3
    assert (_down(device, out)[1] == 0).all() and np.isposinf(_down(device, lse)[1]).all()


@pytest.mark.parametrize("length, room", [(20, 0), (33, 0), (64, 0), (33, 9000), (64, 9000), (33, 40000), (64, 40000)])
@pytest.mark.parametrize("dtype, bits, dim", [("bfloat16", 16, 128), ("float16", 16, 64), ("bfloat16", 4, 128),
                                              ("float16", 4, 64), ("float16", 16, 72)])
def test_attention_rows_do_not_feel_keys_they_do_not_see(device, dtype, bits, dim, length, room):
    """Five query tokens; the third one's key and value are infinite or not a number: the two before
    it are as without them, the others are not numbers."""
    rng = _rng("unseen", dtype, bits, dim, length)
    heads, kv, block, count = 4, 2, 16, 5
    table, sides = _make_cache(device, rng, dtype, bits, [length], kv, dim, block, "head", room=room)
    at = length - 3
    for side in sides:
        if bits == 4:
            par = side[1].read()
            par[table[0, at // block], :, at % block] = np.nan
            side[1].buffer = _up(device, par, dtype)
            side[1].view = _View(side[1].buffer, par.shape)
        else:
            rows = side[0].read()
            rows[table[0, at // block], :, at % block, ::2] = np.inf
            rows[table[0, at // block], :, at % block, 1::2] = np.nan
            side[0].buffer = _up(device, rows, dtype)
            side[0].view = _View(side[0].buffer, rows.shape)
    q = serving.nearest(rng.standard_normal((count, heads, dim)), dtype)
    out, lse = _up(device, np.full(q.shape, 7.0), dtype), _up(device, np.full((count, heads), 7.0), "float32")
    work = device.alloc((ops.attention_paged_workspace(count, heads, kv, dim),), "uint8")
    extra = dict(k_params=sides[0][1].view, v_params=sides[1][1].view) if bits == 4 else {}
    ops.attention_paged(_up(device, q, dtype), sides[0][0].view, sides[1][0].view, device.upload(table),
                        device.upload(np.array([length], np.int32)), out, work, lse=lse, **extra)
    device.check_status()
    got, got_lse = _down(device, out), _down(device, lse)
    k, v = (serving.gather(side[2], table[0], length, block)[:length - 3] for side in sides)
    ref, ref_lse, mass, top = serving.attention_rows(q[:2], k, v, dim ** -0.5, True)
    size = np.abs(v).max() if bits != 4 else 4 * np.abs(v).max()
    bound = size * (2.0 ** -9 + (dim + 16) * 2.0 ** -20 * (1 + top[..., None])) + np.abs(ref) * 2.0 ** -8
    assert (np.abs(got[:2] - ref) <= bound).all() and (np.abs(got_lse[:2] - ref_lse) <= 1e-3 * (1 + top)).all()
    assert np.isnan(got[2:]).all() and np.isnan(got_lse[2:]).all()


def test_attention_spans_outside_the_rows(device):
    """cu_seqlens_q that points behind the rows, or runs backwards, writes nothing outside."""
    rng = _rng("spans")
    table, sides = _make_cache(device, rng, "bfloat16", 16, [40, 40, 40], 1, 64, 16, "head")
    q = serving.nearest(rng.standard_normal((4, 2, 64)), "bfloat16")
    out = _up(device, np.full(q.shape, 7.0), "bfloat16")
    work = device.alloc((ops.attention_paged_workspace(4, 2, 1, 64),), "uint8")
    ops.attention_paged(_up(device, q, "bfloat16"), sides[0][0].view, sides[1][0].view, device.upload(table),
                        device.upload(np.array([40, 40, 40], np.int32)), out, work,
                        cu_seqlens_q=device.upload(np.array([-3, 2, 1, 900], np.int32)))
    device.check_status()
    assert np.isfinite(_down(device, out)).all()


# ------------------------------------------------------------------------------------ int8
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("pad", [5, 8])
@pytest.mark.parametrize("shape", [(1, 1), (3, 67), (5, 128), (33, 4096), (7, 11008), (2, 40000), (6, 520), (5, 16384)])
def test_quantize_rows(device, dtype, shape, pad):
    rng = _rng(dtype, shape)
    x = serving.nearest(rng.standard_normal(shape) * 3, dtype)
    if shape[0] > 4:
        x[1] = 0
        x[2, 0], x[3, -1] = np.inf, np.nan
        # quotients that lie exactly between two codes
        x[4] = serving.nearest((rng.integers(-126, 127, shape[1]) + 0.5), dtype)
        x[4, 0] = 127.0
    wide = np.zeros((shape[0], shape[1] + pad))
    wide[:, :shape[1]] = x
    dx = _View(_up(device, wide, dtype), shape, (shape[1] + pad, 1))
    out, scale = device.alloc(shape, "int8"), device.alloc((shape[0],), "float32")
    ops.quantize_rows(dx, out, scale)
    device.check_status()
    codes, ref = serving.quantize_rows(np.where(np.isfinite(x), x, 0))
    fine = np.isfinite(x).all(1)
    got, got_scale = device.download(out), device.download(scale)
    assert np.array_equal(got_scale[fine], ref[fine]) and not np.isfinite(got_scale[~fine]).any()
    assert np.array_equal(got[fine], codes[fine]) and (got[~fine] == 0).all()


INT8 = [(1, 1, 1), (3, 5, 7), (1, 128, 64), (8, 256, 512), (17, 136, 1040), (33, 96, 100), (64, 1000, 256),
        (129, 257, 272), (128, 128, 16), (300, 520, 1056), (513, 776, 400), (2, 4096, 8192)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("shape", INT8)
@pytest.mark.parametrize("act", ["none", "gelu_tanh"])
def test_linear_int8(device, dtype, shape, act):
    m, n, k = shape
    _check_linear(device, dtype, m, n, k, act, bias="float32" if dtype == "float32" else dtype, pad=0)


def _check_linear(device, dtype, m, n, k, act, bias, pad, stream=0):
    rng = _rng(dtype, m, n, k, act, pad)
    x, w = (rng.integers(-127, 128, (r, k + pad)).astype(np.int8) for r in (m, n))
    sx = rng.uniform(0.5, 1.5, m).astype(np.float32) / 100
    sw = rng.uniform(0.5, 1.5, n).astype(np.float32) / (50 * np.sqrt(k)).astype(np.float32)
    b = serving.nearest(rng.standard_normal(n), bias) if bias else None
    dx, dw = (_View(device.upload(t), (t.shape[0], k), (k + pad, 1)) for t in (x, w))
    y = _up(device, np.full((m, n + pad), 7.0), dtype)
    codes = {"none": abi.ACT_NONE, "gelu_erf": abi.ACT_GELU_ERF, "gelu_tanh": abi.ACT_GELU_TANH,
             "leaky_relu": abi.ACT_LEAKY_RELU}
    ops.linear_int8(dx, device.upload(sx), dw, device.upload(sw), _View(y, (m, n), (n + pad, 1)),
                    bias=_up(device, b, bias) if bias else None, act=codes[act], stream=stream)
    if stream:
        abi.check(abi.lib().b200_stream_sync(stream))
    device.check_status()
    total = x[:, :k].astype(np.float64) @ w[:, :k].astype(np.float64).T
    product = total * sx.astype(np.float64)[:, None] * sw.astype(np.float64)
    z = product + (b if b is not None else 0)
    ref = {"none": lambda t: t, "gelu_erf": oracle.gelu_erf, "gelu_tanh": oracle.gelu_tanh,
           "leaky_relu": oracle.leaky_relu}[act](z)
    # the sum as a float, the scales' product, the fused multiply-add: 3 roundings; the activation's
    # slope is below 1.13 and its own evaluation good to 16 roundings of z (its tail is z * small)
    before = 3 * 2.0 ** -24 * np.abs(product) + 2.0 ** -24 * np.abs(z)
    slack = 1.13 * before + (16 * 2.0 ** -24 * np.abs(z) if act != "none" else 0)
    got = _down(device, y)
    bound = slack + serving.half_step(dtype) * np.abs(ref) * 1.01 + 2.0 ** -25
    bad = ~(np.abs(got[:, :n] - ref) <= bound)
    assert not bad.any(), (np.argwhere(bad)[:4], got[:, :n][bad][:4], ref[bad][:4])
    assert (got[:, n:] == 7).all()


@pytest.mark.parametrize("m, n, k", [(2560, 2048, 64), (4097, 1288, 336), (2305, 2100, 144), (4100, 1283, 160),
                                     (100, 300, 4096), (250, 3000, 2064), (40, 500, 1280)])
@pytest.mark.parametrize("dtype, act, bias", [("bfloat16", "gelu_tanh", "bfloat16"), ("float32", "none", "float16"),
                                              ("float16", "gelu_erf", None)])
def test_linear_int8_tensor_core_tiles(device, dtype, act, bias, m, n, k):
    """Enough 256 x 256 tiles for the CTA pairs, ragged and unaligned outputs; token tiles of 64, 128
    and 256 with K cut between the CTAs of a cluster."""
    _check_linear(device, dtype, m, n, k, act, bias, pad=0)


@pytest.mark.parametrize("act", ["gelu_erf", "leaky_relu"])
@pytest.mark.parametrize("m, n, k, bias, pad", [(5, 64, 96, None, 3), (130, 192, 320, "bfloat16", 16), (4, 72, 64, "float32", 16)])
def test_linear_int8_strides_and_activations(device, act, m, n, k, bias, pad):
    _check_linear(device, "float16", m, n, k, act, bias, pad)


@pytest.mark.parametrize("m, n, k, pad", [(3, 40, 5, 11), (40, 200, 17, 15), (2600, 2048, 24, 8)])
def test_linear_int8_short_sums(device, m, n, k, pad):
    """Fewer columns than a 16-byte row holds, rows on 16-byte boundaries."""
    _check_linear(device, "bfloat16", m, n, k, "none", None, pad)


def test_linear_int8_one_row_for_all(device):
    """x with a row stride of zero, as an expanded tensor has."""
    rng = _rng("expanded")
    x, w = rng.integers(-127, 128, (1, 64)).astype(np.int8), rng.integers(-127, 128, (48, 64)).astype(np.int8)
    y, one = device.alloc((5, 48), "float32"), device.upload(np.ones(48, np.float32))
    ops.linear_int8(_View(device.upload(x), (5, 64), (0, 1)), device.upload(np.ones(5, np.float32)),
                    device.upload(w), one, y)
    device.check_status()
    assert np.array_equal(device.download(y), np.repeat(x.astype(np.float32) @ w.T.astype(np.float32), 5, 0))


def test_linear_int8_activation_far_out(device):
    """GELU where its exponential overflows and where the result vanishes."""
    n = 64
    x, w = np.ones((1, 32), np.int8), np.zeros((n, 32), np.int8)
    w[:, 0] = np.arange(-32, 32)
    for dtype in ("bfloat16", "float32"):
        y = device.alloc((1, n), dtype)
        ops.linear_int8(device.upload(x), device.upload(np.full(1, 100.0, np.float32)), device.upload(w),
                        device.upload(np.ones(n, np.float32)), y, act=abi.ACT_GELU_TANH)
        device.check_status()
        z = np.arange(-32, 32) * 100.0
        assert np.array_equal(_down(device, y)[0], np.where(z > 0, serving.nearest(z, dtype), 0))


def test_linear_int8_largest_sums(device):
    """127 * 127 * K at the largest K: exact beyond 2^24."""
    k = 131056
    x, w = np.full((2, k), 127, np.int8), np.full((3, k), 127, np.int8)
    x[1], w[1] = -127, -128
    y = device.alloc((2, 3), "float32")
    one = device.upload(np.ones(3, np.float32))
    ops.linear_int8(device.upload(x), device.upload(np.ones(2, np.float32)), device.upload(w), one, y)
    device.check_status()
    total = x.astype(np.int64) @ w.astype(np.int64).T
    assert np.array_equal(device.download(y), total.astype(np.float32))


# ----------------------------------------------------------------------- together, captured
def _layer(device, rng, seqs, bits, dim, heads, kv, width, block, dtype):
    """Buffers of one decoder layer's attention half in low precision."""
    hidden = heads * dim
    rows = (heads + 2 * kv) * dim
    s = {"x": serving.nearest(rng.standard_normal((seqs, hidden)), dtype),
         "w_in": rng.integers(-127, 128, (rows, hidden)).astype(np.int8),
         "w_out": rng.integers(-127, 128, (hidden, hidden)).astype(np.int8)}
    s["sw_in"] = (rng.uniform(0.5, 1.5, rows) / (73 * np.sqrt(hidden))).astype(np.float32)
    s["sw_out"] = (rng.uniform(0.5, 1.5, hidden) / (73 * np.sqrt(hidden))).astype(np.float32)
    s["cos"], s["sin"] = _angles(width * block, dim // 2)
    return s


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("bits, dim, heads, kv", [(4, 128, 8, 2), (16, 64, 6, 2)])
def test_a_layer_decodes_token_by_token(device, bits, dim, heads, kv, captured):
    """quantize -> int8 projection -> rotate + append -> attention -> quantize -> int8 projection,
    five steps of a batch; as single launches and as one captured graph whose index tensors
    change between replays, on a stream of its own."""
    dtype, seqs, block, width = "bfloat16", 5, 16, 2
    rng = _rng("layer", bits, dim)
    s = _layer(device, rng, seqs, bits, dim, heads, kv, width, block, dtype)
    hidden, rows = heads * dim, (heads + 2 * kv) * dim
    d = {n: device.upload(s[n]) for n in ("w_in", "w_out", "sw_in", "sw_out", "cos", "sin")}
    x = _up(device, s["x"], dtype)
    pages = seqs * width
    table = rng.permutation(pages).reshape(seqs, width).astype(np.int32)
    d_table = device.upload(table)
    row = dim if bits == 16 else dim // 2
    zero = np.zeros((pages, kv, block, row), np.uint8 if bits == 4 else np.float64)
    caches = [Paged(device, zero, "uint8" if bits == 4 else dtype, "token") for _ in range(2)]
    params = [Paged(device, np.zeros((pages, kv, block, 2)), dtype, "token") for _ in range(2)] if bits == 4 else None
    extra = dict(k_params=params[0].view, v_params=params[1].view) if params else {}
    buf = {"x8": device.alloc((seqs, hidden), "int8"), "sx": device.alloc((seqs,), "float32"),
           "qkv": device.alloc((seqs, rows), dtype), "q": device.alloc((seqs, heads, dim), dtype),
           "o": device.alloc((seqs, heads, dim), dtype), "y": device.alloc((seqs, hidden), dtype),
           "work": device.alloc((ops.attention_paged_workspace(seqs, heads, kv, dim),), "uint8"),
           "seq": device.upload(np.arange(seqs, dtype=np.int32)),
           "pos": device.alloc((seqs,), "int32"), "len": device.alloc((seqs,), "int32")}

    def part(first, count):
        return _View(buf["qkv"], (seqs, count, dim), (rows, dim, 1), offset=first * dim)

    def step(stream):
        ops.quantize_rows(x, buf["x8"], buf["sx"], stream=stream)
        ops.linear_int8(buf["x8"], buf["sx"], d["w_in"], d["sw_in"], buf["qkv"], stream=stream)
        ops.kv_append(part(heads, kv), part(heads + kv, kv), caches[0].view, caches[1].view, d_table, buf["seq"],
                      buf["pos"], cos=d["cos"], sin=d["sin"], q=part(0, heads), q_out=buf["q"], stream=stream, **extra)
        ops.attention_paged(buf["q"], caches[0].view, caches[1].view, d_table, buf["len"], buf["o"], buf["work"],
                            stream=stream, **extra)
        ops.quantize_rows(_View(buf["o"], (seqs, hidden)), buf["x8"], buf["sx"], stream=stream)
        ops.linear_int8(buf["x8"], buf["sx"], d["w_out"], d["sw_out"], buf["y"], stream=stream)

    stream = graph.Stream() if captured else None
    g = None
    first = rng.integers(0, 12, seqs)
    held = [[[] for _ in range(seqs)] for _ in range(2)]
    for n in range(5):
        pos = (first * 0 + n).astype(np.int32)
        device.copy_in(buf["pos"], pos, sync=True)
        device.copy_in(buf["len"], pos + 1, sync=True)
        if not captured:
            step(0)
        else:
            if g is None:
                step(stream.handle)  # once outside the capture
                stream.synchronize()
                with graph.capture(stream) as g:
                    step(stream.handle)
            g.launch(stream)
            stream.synchronize()
        device.check_status()
        qkv = _down(device, buf["qkv"]).reshape(seqs, heads + 2 * kv, dim)
        codes, scale = serving.quantize_rows(s["x"])
        ref = (codes.astype(np.float64) @ s["w_in"].astype(np.float64).T) * scale.astype(np.float64)[:, None] * s["sw_in"]
        assert (np.abs(qkv.reshape(seqs, rows) - ref) <= np.abs(ref) * (serving.half_step(dtype) + 2.0 ** -21)).all()
        c, si = s["cos"][pos], s["sin"][pos]
        q = serving.nearest(serving.rotate(qkv[:, :heads], c, si), dtype)
        assert np.array_equal(_down(device, buf["q"]), q)
        k = serving.nearest(serving.rotate(qkv[:, heads:heads + kv], c, si), dtype)
        for side, new in ((0, k), (1, qkv[:, heads + kv:])):
            if bits == 4:
                new = serving.stands_for(*serving.four_bits(new, dtype))
            for z in range(seqs):
                held[side][z].append(new[z])
        got = _down(device, buf["o"])
        for z in range(seqs):
            k_z, v_z = np.stack(held[0][z]), np.stack(held[1][z])
            out, _, mass, top = serving.attention_rows(q[z:z + 1], k_z, v_z, dim ** -0.5, True)
            # rows of few keys: the bound of the module's head, with twice |v| for low + 15 scale
            size = 4 * np.abs(v_z).max() + 1
            bound = np.abs(out[0]) * 2.0 ** -8 + size * (2.0 ** -9 + (dim + 16) * 2.0 ** -20 * (1 + top[0][:, None]))
            assert (np.abs(got[z] - out[0]) <= bound).all()
        codes, scale = serving.quantize_rows(got.reshape(seqs, hidden))
        ref = (codes.astype(np.float64) @ s["w_out"].astype(np.float64).T) * scale.astype(np.float64)[:, None] * s["sw_out"]
        assert (np.abs(_down(device, buf["y"]) - ref) <= np.abs(ref) * (serving.half_step(dtype) + 2.0 ** -21)).all()
        # the next step's input
        x_next = serving.nearest(rng.standard_normal((seqs, hidden)), dtype)
        s["x"] = x_next
        device.copy_in(x, (x_next.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16), sync=True)
    if stream is not None:
        g.close()
        stream.close()


@pytest.mark.parametrize("bits", [16, 4])
def test_graphs_with_a_workspace_each_replay_side_by_side(device, bits):
    """Two captured calls over contexts that are cut between CTAs, replayed many times at once on two
    streams: the results of single launches, bit for bit, whatever the workspaces held before."""
    rng = _rng("graphs", bits)
    dtype, block, lengths, heads, kv, dim = "bfloat16", 16, [3000, 1700, 20], 8, 2, 128
    table, sides = _make_cache(device, rng, dtype, bits, lengths, kv, dim, block, "head", room=40000)
    extra = dict(k_params=sides[0][1].view, v_params=sides[1][1].view) if bits == 4 else {}
    d_table, d_len = device.upload(table), device.upload(np.array(lengths, np.int32))
    size = ops.attention_paged_workspace(3, heads, kv, dim)
    calls = []
    for i in range(2):
        q = _up(device, serving.nearest(rng.standard_normal((3, heads, dim)), dtype), dtype)
        out, lse = device.alloc((3, heads, dim), dtype), device.alloc((3, heads), "float32")
        work = device.upload(rng.integers(0, 256, size).astype(np.uint8))

        def run(stream, q=q, out=out, lse=lse, work=work):
            ops.attention_paged(q, sides[0][0].view, sides[1][0].view, d_table, d_len, out, work, lse=lse,
                                stream=stream, **extra)
        run(0)
        device.synchronize()
        calls.append((run, out, lse, device.download(out).copy(), device.download(lse).copy()))
    streams = [graph.Stream() for _ in calls]
    graphs = []
    for (run, *_), stream in zip(calls, streams):
        with graph.capture(streams[0]) as g:   # captured on one stream, replayed on two
            run(streams[0].handle)
        graphs.append(g)
    for _ in range(20):
        for g, stream in zip(graphs, streams):
            g.launch(stream)
    for stream in streams:
        stream.synchronize()
    device.check_status()
    for _, out, lse, expected, expected_lse in calls:
        assert np.array_equal(device.download(out), expected) and np.array_equal(device.download(lse), expected_lse)
    for g in graphs:
        g.close()
    for stream in streams:
        stream.close()


def test_handles_through_the_launch_surface(device):
    """The same operators as registered kernels of the device protocol, launched twice (the
    second launch replays the recorded calls)."""
    rng = _rng("handles")
    t, heads, kv, dim, block = 4, 4, 2, 64, 16
    table = np.array([[1, 0]], np.int32)
    q, k, v = (serving.nearest(rng.standard_normal((t, h, dim)), "float16") for h in (heads, kv, kv))
    cos, sin = _angles(t, dim // 2)
    dq, dk, dv = (_up(device, a, "float16") for a in (q, k, v))
    caches = [Paged(device, np.zeros((2, kv, block, dim // 2), np.uint8), "uint8", "head") for _ in range(2)]
    params = [Paged(device, np.zeros((2, kv, block, 2)), "float16", "head") for _ in range(2)]
    q_out, out, lse = device.alloc(q.shape, "float16"), device.alloc(q.shape, "float16"), device.alloc((t, heads), "float32")
    shared = {"k_cache_ptr": caches[0].buffer, "v_cache_ptr": caches[1].buffer, "k_params_ptr": params[0].buffer,
              "v_params_ptr": params[1].buffer, "page_table_ptr": device.upload(table), "T": t, "Z": 1, "WIDTH": 2,
              "H": heads, "H_KV": kv, "HEAD_DIM": dim, "PAGES": 2, "BLOCK": block, "BITS": 4}
    append = {"k_ptr": dk, "v_ptr": dv, "seq_ptr": device.upload(np.zeros(t, np.int32)),
              "pos_ptr": device.upload(np.arange(t, dtype=np.int32)), "cos_ptr": device.upload(cos),
              "sin_ptr": device.upload(sin), "q_ptr": dq, "q_out_ptr": q_out, "ROT_DIM": dim, "ANGLES": t,
              "INTERLEAVED": False, **shared}
    attend = {"q_ptr": q_out, "lengths_ptr": device.upload(np.array([t], np.int32)), "cu_seqlens_q_ptr": None,
              "out_ptr": out, "lse_ptr": lse, "scale": dim ** -0.5, "CAUSAL": True, **shared}
    for _ in range(2):
        for kernel, values, grid in ((kernels.kv_append_kernel, append, (t,)),
                                     (kernels.paged_attention_kernel, attend, (t, heads))):
            positional, keywords = harness.bind_arguments(kernel, values)
            device.launch(kernel, grid, positional, keywords)
    device.synchronize()
    assert np.array_equal(_down(device, q_out), serving.nearest(serving.rotate(q, cos, sin), "float16"))
    k4 = serving.stands_for(*serving.four_bits(serving.nearest(serving.rotate(k, cos, sin), "float16"), "float16"))
    v4 = serving.stands_for(*serving.four_bits(v, "float16"))
    ref, ref_lse, _, _ = serving.attention_rows(_down(device, q_out), k4, v4, dim ** -0.5, True)
    assert np.abs(_down(device, out) - ref).max() <= 2.0 ** -9 * 4 * np.abs(v4).max()
    assert np.abs(_down(device, lse) - ref_lse).max() <= 1e-4
    # the linear layer's pair
    m, n, kk = 3, 32, 64
    x = serving.nearest(rng.standard_normal((m, kk)), "float16")
    w, sw = rng.integers(-127, 128, (n, kk)).astype(np.int8), np.full(n, 0.01, np.float32)
    x8, sx, y = device.alloc((m, kk), "int8"), device.alloc((m,), "float32"), device.alloc((m, n), "float32")
    device.launch(kernels.quantize_rows_kernel, (m,), [_up(device, x, "float16"), x8, sx, m, kk], {})
    device.launch(kernels.linear_int8_kernel, (1,), [x8, sx, device.upload(w), device.upload(sw), None, y, m, n, kk, 0], {})
    device.synchronize()
    codes, scale = serving.quantize_rows(x)
    assert np.array_equal(device.download(x8), codes)
    ref = (codes.astype(np.float64) @ w.T.astype(np.float64)) * scale.astype(np.float64)[:, None] * sw.astype(np.float64)
    assert np.allclose(device.download(y), ref, rtol=2.0 ** -21, atol=0)


def test_memory_that_the_launch_cannot_reach_is_refused(device):
    """Pageable host memory in the place of device memory."""
    host = np.zeros((4, 64), np.float16)

    class Host:
        shape, dtype = host.shape, "float16"

        @staticmethod
        def data_ptr():
            return host.ctypes.data

    with pytest.raises(abi.B200Error) as err:
        ops.quantize_rows(Host, device.alloc((4, 64), "int8"), device.alloc((4,), "float32"))
    assert err.value.status == abi.REJECTED
    # page-locked memory reaches the row kernels, not the copies of the tensor-core ones
    pinned = device.pinned_empty((4, 64), np.float16)
    pinned.array[:] = np.arange(64)
    out, scale = device.alloc((4, 64), "int8"), device.alloc((4,), "float32")

    class Locked:
        shape, dtype = (4, 64), "float16"

        @staticmethod
        def data_ptr():
            return pinned.ptr

    ops.quantize_rows(Locked, out, scale)
    device.synchronize()
    assert np.array_equal(device.download(out), serving.quantize_rows(np.asarray(pinned.array, np.float64))[0])
    Locked.dtype = "int8"
    with pytest.raises(abi.B200Error) as err:
        ops.linear_int8(Locked, scale, out, scale, device.alloc((4, 4), "float32"))
    assert err.value.status == abi.REJECTED
    device.synchronize()


@pytest.mark.parametrize("bits", [16, 4])
def test_attention_with_unlike_strides_of_keys_and_values(device, bits):
    """K pages head-major, V pages token-major: the kernel that takes any strides."""
    rng = _rng("unlike", bits)
    dtype, block, lengths = "float16", 16, [40, 9]
    table, sides = _make_cache(device, rng, dtype, bits, lengths, 2, 64, block, "head")
    values = sides[1][0].read() if bits == 4 else None
    other = Paged(device, values if bits == 4 else np.nan_to_num(sides[1][0].read(), nan=0, posinf=0),
                  "uint8" if bits == 4 else dtype, "token")
    q = serving.nearest(rng.standard_normal((2, 4, 64)), dtype)
    out, lse = device.alloc(q.shape, dtype), device.alloc((2, 4), "float32")
    work = device.alloc((ops.attention_paged_workspace(2, 4, 2, 64),), "uint8")
    extra = dict(k_params=sides[0][1].view, v_params=sides[1][1].view) if bits == 4 else {}
    ops.attention_paged(_up(device, q, dtype), sides[0][0].view, other.view, device.upload(table),
                        device.upload(np.array(lengths, np.int32)), out, work, lse=lse, **extra)
    device.check_status()
    _check_attention(device, dtype, q, out, lse, table, sides, lengths, [(0, 1), (1, 2)], 0.125, True, block)
