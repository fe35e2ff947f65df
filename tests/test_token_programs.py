"""The token side of a language model: `gather`, `scatter_add`, `token_log_prob` and the losses of
`accy_b200.nn`, as recorded programs.

CPU: types, refusals, wire bytes, derived programs (the oracle evaluates them; gradients against
central differences in f64), shard analysis, and what the planner makes of them.  GPU: every
operation against a numpy evaluation in f64 at the sizes and values where it can go wrong.

Tolerances count roundings: half a step of a type is U[dtype] relative to the value.  Device sums are
held in f32, so a sum of n terms is off by at most n * U["f32"] * sum(|terms|) before its one
rounding to the result's type.
"""
import ctypes
import struct

import numpy as np
import pytest

from accy_b200 import nn, synthetic, tensor
from accy_b200._native import lib
from oracle import oracle

T = tensor
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24, "f64": 2.0 ** -53}
TINY = {"bf16": 2.0 ** -133, "f16": 2.0 ** -24, "f32": 2.0 ** -126, "f64": 2.0 ** -1022}  # below: subnormal steps or flushed
NP = {"bf16": np.uint16, "f16": np.float16, "f32": np.float32, "f64": np.float64, "i8": np.int8, "i16": np.int16, "i32": np.int32,
      "i64": np.int64, "u8": np.uint8, "u16": np.uint16, "u32": np.uint32, "u64": np.uint64}


def stored(dtype, x):
    """f64 values -> the array of the element type that holds them"""
    return synthetic.f32_to_bf16_bits(np.asarray(x, np.float32)) if dtype == "bf16" else np.asarray(x).astype(NP[dtype])


def exactly(dtype, a):
    """the f64 values an array of the element type holds"""
    return synthetic.bf16_bits_to_f32(a).astype(np.float64) if dtype == "bf16" else np.asarray(a, np.float64)


def shape_of(t):
    return tuple(e for _, e in t.dims)


def run(session, program, inputs):
    compiled = session.compile(program)
    outs = [np.full(shape_of(t), 77).astype(NP[t.dtype]) for t in program.output_types]
    session.invoke(compiled, inputs, outs)
    session.release(compiled)
    return [exactly(t.dtype, o) for t, o in zip(program.output_types, outs)]


def close(got, want, allowed):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    odd = ~np.isfinite(want)
    assert np.array_equal(got[odd & ~np.isnan(want)], want[odd & ~np.isnan(want)])
    off = np.where(odd, 0, np.abs(np.where(odd, 0, got) - np.where(odd, 0, want)))
    allowed = np.broadcast_to(np.where(np.isfinite(allowed), allowed, 0), off.shape)
    worst = int(np.argmax(off - allowed)) if off.size else 0
    assert off.size == 0 or np.all(off <= allowed), (np.unravel_index(worst, off.shape), got.reshape(-1)[worst], want.reshape(-1)[worst])


def lookup(x, idx, axis):
    """x with `axis` replaced by the axes of idx, in f64; zeros for a number outside"""
    rows = np.moveaxis(x, axis, 0)
    out = np.zeros(idx.shape + rows.shape[1:])
    for at in np.ndindex(*idx.shape):
        if 0 <= idx[at] < len(rows):
            out[at] = rows[int(idx[at])]
    return np.moveaxis(out, list(range(idx.ndim)), list(range(axis, axis + idx.ndim)))


def scattered(base, idx, up, axis):
    """(sum, sum of magnitudes, number of terms) in f64"""
    out, mag, n = np.moveaxis(base.copy(), axis, 0), np.moveaxis(np.abs(base), axis, 0).copy(), np.ones(base.shape[axis])
    rows = np.moveaxis(up, list(range(axis, axis + idx.ndim)), list(range(idx.ndim))).reshape((idx.size,) + out.shape[1:])
    known = (idx.reshape(-1) >= 0) & (idx.reshape(-1) < base.shape[axis])
    at = idx.reshape(-1)[known].astype(np.int64)
    np.add.at(out, at, rows[known])
    np.add.at(mag, at, np.abs(rows[known]))
    np.add.at(n, at, 1)
    terms = n.reshape((-1,) + (1,) * (base.ndim - 1))
    return np.moveaxis(out, 0, axis), np.moveaxis(mag, 0, axis), np.moveaxis(np.broadcast_to(terms, out.shape), 0, axis)


def log_prob_of(x, tok):
    """(log p, p, one-hot, known) along the last axis, in f64"""
    known = (tok >= 0) & (tok < x.shape[-1])
    at = np.where(known, tok, 0).astype(np.int64)[..., None]
    with np.errstate(all="ignore"):
        shifted = x - x.max(-1, keepdims=True)
        e = np.exp(shifted)
        log_p = np.take_along_axis(shifted, at, -1)[..., 0] - np.log(e.sum(-1))
        p = e / e.sum(-1, keepdims=True)
    hot = np.zeros_like(x)
    np.put_along_axis(hot, at, known[..., None].astype(x.dtype), -1)
    return np.where(known, log_p, 0), p, hot, known


def spread_of(x):
    """the largest finite distance of a logit that matters (p >= 2^-60) from its row's maximum"""
    with np.errstate(all="ignore"):
        d = np.where(np.isfinite(x), x.max(-1, keepdims=True) - x, 0)
    d = np.where(np.isfinite(d), d, 0)
    return float(np.minimum(d, 42.0).max()) if d.size else 0.0


def p_error(x):
    """Relative error of a probability: its exponent (x - m) * log2(e) takes three roundings (difference,
    product, constant) of at most 42 * log2(e) where p >= 2^-60; 2^-22 for the exponential and as much for
    those in the sum; the sum is folded by threads of at most 64 terms, then in trees of at most 13 levels."""
    return 3 * U["f32"] * spread_of(x) + 2 * 2.0 ** -22 + 80 * U["f32"]


# ---------------------------------------------------------------------------------------------
# recording, wire bytes, refusals
# ---------------------------------------------------------------------------------------------
def refused(name, body, *specs):
    with pytest.raises(T.TensorError) as e:
        T.define("refused", list(specs), body)
    assert e.value.name == name


TABLE, IDS = T.spec("bf16", vocab=11, dim=6), T.spec("i32", batch=2, seq=3)
LOGITS = T.spec("bf16", batch=2, seq=3, vocab=11)


def test_types_of_the_operations():
    p = T.define("g", [TABLE, IDS], lambda b, a: a[0].gather(a[1], "vocab"))
    assert repr(p.output_types[0]) == "bf16[batch=2, seq=3, dim=6]"
    p = T.define("g", [TABLE, IDS], lambda b, a: a[0].gather(a[1], "dim"))
    assert repr(p.output_types[0]) == "bf16[vocab=11, batch=2, seq=3]"
    p = T.define("s", [TABLE, IDS, T.spec("bf16", dim=6)], lambda b, a: a[0].scatter_add(a[1], a[2], "vocab"))
    assert repr(p.output_types[0]) == "bf16[vocab=11, dim=6]"
    p = T.define("l", [LOGITS, T.spec("u8", seq=3, batch=2)], lambda b, a: a[0].token_log_prob(a[1], "vocab"))
    assert repr(p.output_types[0]) == "f32[batch=2, seq=3]"
    p = T.define("e", [IDS, T.spec("f16", batch=2, seq=3, dim=6)], lambda b, a: nn.embedding_grad(a[0], a[1], "vocab", 11, scale=2.0))
    assert repr(p.output_types[0]) == "f16[vocab=11, dim=6]"


def test_recording_refusals():
    floats, mask = T.spec("f32", batch=2, seq=3), T.spec("i1", batch=2, seq=3)
    refused("AxisNotFound", lambda b, a: a[0].gather(a[1], "nope"), TABLE, IDS)
    refused("NonIntegerDType", lambda b, a: a[0].gather(a[1], "vocab"), TABLE, floats)
    refused("NonIntegerDType", lambda b, a: a[0].gather(a[1], "vocab"), TABLE, mask)
    refused("DuplicateAxis", lambda b, a: a[0].gather(a[1], "vocab"), T.spec("f32", vocab=11, seq=6), IDS)
    refused("AxisNotFound", lambda b, a: a[0].scatter_add(a[1], a[2], "nope"), TABLE, IDS, TABLE)
    refused("DTypeMismatch", lambda b, a: a[0].scatter_add(a[1], a[2], "vocab"), TABLE, IDS, T.spec("f32", batch=2, seq=3, dim=6))
    refused("NonFloatDType", lambda b, a: a[0].scatter_add(a[1], a[2], "vocab"), T.spec("i32", vocab=11), IDS, IDS)
    refused("NonIntegerDType", lambda b, a: a[0].scatter_add(a[1], a[2], "vocab"), TABLE, floats, T.spec("bf16", dim=6))
    refused("AxisExtentMismatch", lambda b, a: a[0].scatter_add(a[1], a[2], "vocab"), TABLE, IDS, T.spec("bf16", batch=2, seq=4, dim=6))
    refused("AxisNotFound", lambda b, a: a[0].token_log_prob(a[1], "nope"), LOGITS, IDS)
    refused("NonFloatDType", lambda b, a: a[0].token_log_prob(a[1], "vocab"), T.spec("f64", batch=2, seq=3, vocab=5), IDS)
    refused("NonIntegerDType", lambda b, a: a[0].token_log_prob(a[1], "vocab"), LOGITS, floats)
    refused("AxisExtentMismatch", lambda b, a: a[0].token_log_prob(a[1], "vocab"), LOGITS, T.spec("i32", batch=2, seq=4))
    refused("AxisNotFound", lambda b, a: a[0].token_log_prob(a[1], "vocab"), LOGITS, T.spec("i32", batch=2, seq=3, other=4))
    refused("AxisNotFound", lambda b, a: nn.cross_entropy(a[0], a[1], "nope"), LOGITS, IDS)
    refused("NonIntegerDType", lambda b, a: nn.cross_entropy(a[0], a[1], "vocab"), LOGITS, floats)
    with pytest.raises(T.TensorError):   # a value of another recording
        other = []
        T.define("other", [IDS], lambda b, a: other.append(a[0]) or a[0])
        T.define("cross", [TABLE], lambda b, a: a[0].gather(other[0], "vocab"))


def reencode(wire):
    src = ctypes.create_string_buffer(bytes(wire), len(wire))
    out, n, err = ctypes.create_string_buffer(len(wire) + 4096), ctypes.c_size_t(), ctypes.create_string_buffer(256)
    status = lib.accy_b200_wire_reencode(ctypes.cast(src, ctypes.c_void_p), len(wire), ctypes.cast(out, ctypes.c_void_p), len(out),
                                         ctypes.byref(n), ctypes.cast(err, ctypes.c_void_p), 256)
    return status, err.value.decode(), out.raw[:n.value]


def policy_program(dtype="f32", index="i32", batch=2, seq=3, vocab=11, kl=0.05):
    row = T.spec("f32", batch=batch, seq=seq)
    return T.define("policy", [T.spec(dtype, batch=batch, seq=seq, vocab=vocab), T.spec(index, batch=batch, seq=seq), row, row,
                               T.spec("f32", batch=batch), row],
                    lambda b, a: nn.policy_loss(a[0], a[1], "vocab", old=a[2], reference=a[3], advantage=a[4], mask=a[5], clip=0.2, kl=kl))


def test_wire_bytes_round_trip_and_untrusted_types():
    def body(b, a):
        rows = a[0].gather(a[1], "vocab")
        return a[0].scatter_add(a[1], rows, "vocab"), a[2].token_log_prob(a[1], "vocab")
    for program in (T.define("all", [TABLE, IDS, LOGITS], body), policy_program().value_and_grad([0])):
        status, _, again = reencode(program.wire)
        assert status == 0 and again == program.wire
        n, text = ctypes.c_size_t(), ctypes.create_string_buffer(1 << 16)
        src = ctypes.create_string_buffer(program.wire, len(program.wire))
        assert lib.accy_b200_wire_describe(ctypes.cast(src, ctypes.c_void_p), len(program.wire), ctypes.cast(text, ctypes.c_void_p), len(text), ctypes.byref(n)) == 0
        assert text.value.decode() == oracle.describe(program.wire)
    wire = T.define("call", [LOGITS, IDS], lambda b, a: a[0].token_log_prob(a[1], "vocab")).wire
    assert reencode(wire.replace(b"token_log_prob", b"token_log_prog"))[1] == "CustomCallUnsupported"
    at = wire.index(b"accy_b200.token_log_prob") + len(b"accy_b200.token_log_prob")
    assert struct.unpack("<I", wire[at:at + 4]) == (1,)
    assert reencode(wire[:at] + struct.pack("<I", 2) + wire[at + 4:])[1] == "CustomCallUnsupported"
    # the call declares its result as f32: declared as f16 it is refused
    kind = wire.index(b"accy_b200.token_log_prob") - 4
    declared = wire.rindex(struct.pack("<II", 11, 2), 0, kind)
    assert reencode(wire[:declared] + struct.pack("<I", 9) + wire[declared + 4:])[1] == "InvalidProgram"
    # an axis outside the operand
    wire = T.define("g", [TABLE, IDS], lambda b, a: a[0].gather(a[1], "vocab")).wire
    at = wire.rindex(struct.pack("<IIIq", 10, 0, 1, 0)) + 12
    assert reencode(wire[:at] + struct.pack("<q", 2) + wire[at + 8:])[1] == "AxisOutOfRange"


# ---------------------------------------------------------------------------------------------
# derived programs, evaluated by the oracle
# ---------------------------------------------------------------------------------------------
def small_inputs(seed=0):
    rng = np.random.default_rng(seed)
    logits, tok = rng.standard_normal((2, 3, 11)).astype(np.float32), np.array([[3, 10, 0], [7, -1, 2]], np.int32)
    now = log_prob_of(logits.astype(np.float64), tok)[0]
    return [logits, tok, (now - 0.3 * rng.standard_normal((2, 3))).astype(np.float32), (now + rng.standard_normal((2, 3))).astype(np.float32),
            np.array([1.5, -0.7], np.float32), np.array([[1, 1, 0], [1, 1, 1]], np.float32)]


def head_loss(b, a):
    """embedding, a tanh, logits against the same table, cross entropy: the table is looked up and contracted"""
    table, tok, nxt = a
    hidden = nn.embedding(table, tok, "vocab", scale=2.0).tanh()
    return nn.cross_entropy(hidden.contract(table, "dim"), nxt, "vocab")


def head_program(dtype="f32", batch=2, seq=3, vocab=11, dim=6):
    return T.define("head", [T.spec(dtype, vocab=vocab, dim=dim), T.spec("i32", batch=batch, seq=seq), T.spec("i32", batch=batch, seq=seq)], head_loss)


def head_inputs(batch=2, seq=3, vocab=11, dim=6, seed=3):
    rng = np.random.default_rng(seed)
    tok, nxt = (rng.integers(-1, vocab, (batch, seq)).astype(np.int32) for _ in range(2))
    return [(0.5 * rng.standard_normal((vocab, dim))).astype(np.float32), tok, nxt]


def differences(program, inputs, index, wrt_grad, picks=24, seed=5):
    """central differences of a scalar program in f64 against its gradient, at some elements"""
    rng = np.random.default_rng(seed)
    base = [np.asarray(x) for x in inputs]
    for flat in rng.choice(base[index].size, min(picks, base[index].size), replace=False):
        at, h = np.unravel_index(flat, base[index].shape), 2.0 ** -10   # representable next to f32 inputs of this size
        ends = []
        for sign in (1, -1):
            moved = base[index].copy()
            moved[at] += sign * h
            width = moved[at]
            ends.append((float(oracle.run(program.wire, base[:index] + [moved] + base[index + 1:], mode="f64")[0].reshape(-1)[0]), float(width)))
        slope = (ends[0][0] - ends[1][0]) / (ends[0][1] - ends[1][1])
        # third derivatives of these programs are below 200: the difference is off by at most h^2 / 6 times that
        assert abs(slope - wrt_grad[at]) <= 200 * h * h / 6 + 1e-9, (at, slope, wrt_grad[at])


@pytest.mark.parametrize("name", ["cross_entropy", "policy", "head"])
def test_gradients_match_differences(name):
    if name == "head":
        program, inputs = head_program(), head_inputs()
    elif name == "policy":
        program, inputs = policy_program(), small_inputs()
    else:
        program = T.define("ce", [T.spec("f32", batch=2, seq=3, vocab=11), IDS], lambda b, a: nn.cross_entropy(a[0], a[1], "vocab"))
        inputs = small_inputs()[:2]
    value, grad = oracle.run(program.value_and_grad([0]).wire, inputs, mode="f64")
    assert abs(float(value.reshape(-1)[0]) - float(oracle.run(program.wire, inputs, mode="f64")[0].reshape(-1)[0])) < 1e-12
    differences(program, inputs, 0, grad)


def test_gradients_with_respect_to_the_other_inputs_of_the_policy_loss():
    """The advantage is one number per sequence, stretched over its tokens: its gradient sums over them."""
    program, inputs = policy_program(), small_inputs()
    grads = oracle.run(program.grad([2, 3, 4]).wire, inputs, mode="f64")
    for index, grad in zip((2, 3, 4), grads):
        differences(program, inputs, index, grad)
    assert grads[0][0, 2] == 0 and grads[1][0, 2] == 0 and grads[0][1, 1] == 0   # masked, and a token outside


def test_token_types_and_vocabularies_at_their_ends():
    """Losses record for every token type, also where the vocabulary is as large as the type or empty."""
    for dtype, extent in (("u8", 256), ("u8", 255), ("i8", 128), ("i8", 5), ("u8", 0), ("u64", 3)):
        specs = [T.spec("f32", n=4, v=extent), T.spec(dtype, n=4)]
        program = T.define("ce", specs, lambda b, a: nn.cross_entropy(a[0], a[1], "v"))
        tok = np.array([0, 3, 127, 4], NP[dtype])
        x = np.random.default_rng(1).standard_normal((4, extent)).astype(np.float32)
        want = 0.0
        if extent:
            log_p, _, _, known = log_prob_of(x.astype(np.float64), tok)
            want = -log_p.sum() / max(known.sum(), 1)
            assert abs(float(oracle.run(program.wire, [x, tok], mode="f64")[0].reshape(-1)[0]) - want) < 1e-12


def test_gradient_of_scatter_add_and_repeated_lookups():
    def body(b, a):
        base, idx, up, weight = a
        out = base.scatter_add(idx, up, "v")
        again = out.gather(idx, "v").mul(out.gather(idx, "v"))
        return out.mul(weight).sum(["v", "d"]).add(again.sum(["n", "d"]))
    specs = [T.spec("f32", v=5, d=3), T.spec("i32", n=7), T.spec("f32", n=7, d=3), T.spec("f32", v=5, d=3)]
    rng = np.random.default_rng(1)
    inputs = [rng.standard_normal((5, 3)).astype(np.float32), np.array([1, 4, 1, -1, 5, 0, 1], np.int32),
              rng.standard_normal((7, 3)).astype(np.float32), rng.standard_normal((5, 3)).astype(np.float32)]
    program = T.define("scatter", specs, body)
    grads = oracle.run(program.grad([0, 2]).wire, inputs, mode="f64")
    differences(program, inputs, 0, grads[0])
    differences(program, inputs, 2, grads[1])
    assert np.all(grads[1][[3, 4]] == 0)   # numbers outside the axis
    # forward mode against the gradient
    along = [rng.standard_normal(x.shape).astype(np.float32) for x in (inputs[0], inputs[2])]
    value, slope = oracle.run(program.jvp([0, 2]).wire, inputs + along, mode="f64")
    want = sum(float((g * d).sum()) for g, d in zip(grads, along))
    assert abs(float(slope.reshape(-1)[0]) - want) <= 1e-10 * max(1, abs(want))


def test_forward_mode_of_a_log_probability():
    program = T.define("l", [T.spec("f32", batch=2, seq=3, vocab=11), IDS], lambda b, a: a[0].token_log_prob(a[1], "vocab"))
    logits, tok = small_inputs()[:2]
    direction = np.random.default_rng(2).standard_normal(logits.shape).astype(np.float32)
    _, slope = oracle.run(program.jvp([0]).wire, [logits, tok, direction], mode="f64")
    _, p, hot, known = log_prob_of(logits.astype(np.float64), tok)
    assert np.allclose(slope, ((hot - p) * known[..., None] * direction).sum(-1), rtol=0, atol=1e-12)
    with pytest.raises(T.TensorError) as e:   # the sum over 16-bit products would not be f32
        T.define("l", [LOGITS, IDS], lambda b, a: a[0].token_log_prob(a[1], "vocab")).jvp([0])
    assert e.value.name == "UnsupportedDerivative"


def test_second_derivatives_are_refused():
    first = T.define("ce", [T.spec("f32", n=3, vocab=5), T.spec("i32", n=3)], lambda b, a: nn.cross_entropy(a[0], a[1], "vocab")).grad([0])
    assert oracle.run(first.wire, [np.zeros((3, 5), np.float32), np.zeros(3, np.int32)])[0].shape == (3, 5)
    # <gradient, gradient> cannot be recorded on top of a derived program, but forward mode over it can be asked for
    with pytest.raises(T.TensorError) as e:
        first.jvp([0])
    assert e.value.name == "UnsupportedDerivative"


@pytest.mark.parametrize("in_axes", [[0, None], [None, 0], [0, 0], [1, 2], [2, 1]])
@pytest.mark.parametrize("op", ["gather", "scatter_add", "log_prob"])
def test_vmap_equals_the_program_run_once_per_instance(op, in_axes):
    rng = np.random.default_rng(7)
    v, n, d, size = 5, 4, 3, 6

    def body(b, a):
        if op == "gather":
            return a[0].gather(a[1], "v")
        if op == "scatter_add":
            return a[0].scatter_add(a[1], a[0].gather(a[1], "v").mul(b.scalar("f32", 2.0)), "v")
        return a[0].token_log_prob(a[1].rename("n", "d"), "v")
    n = d if op == "log_prob" else n
    program = T.define("one", [T.spec("f32", v=v, d=d), T.spec("i32", n=n)], body)
    if op != "log_prob" and in_axes == [1, 2]:
        in_axes = [1, 1]
    if op == "log_prob" and in_axes[1] == 2:
        in_axes = [1, 1]
    shapes = [(v, d), (n,)]
    full = []
    for shape, axis, kind in zip(shapes, in_axes, "fi"):
        dims = list(shape)
        if axis is not None:
            dims.insert(min(axis, len(dims)), size)
        full.append(rng.standard_normal(dims).astype(np.float32) if kind == "f" else rng.integers(-2, v + 2, dims).astype(np.int32))
    in_axes = [None if a is None else min(a, len(s)) for a, s in zip(in_axes, shapes)]
    mapped = program.vmap(size, in_axes)
    got = oracle.run(mapped.wire, full, mode="f64")[0]
    for i in range(size):
        one = [x if a is None else np.ascontiguousarray(np.take(x, i, a)) for x, a in zip(full, in_axes)]
        assert np.array_equal(got[i], oracle.run(program.wire, one, mode="f64")[0])


def test_vmap_refusals():
    table, ids = T.spec("f32", d=3, v=100), T.spec("u8", n=4)
    with pytest.raises(T.TensorError) as e:   # both mapped, and the axis is not the first
        T.define("g", [table, ids], lambda b, a: a[0].gather(a[1], "v")).vmap(6, [0, 0])
    assert e.value.name == "UnsupportedBatching"
    first = T.define("g", [T.spec("f32", v=100, d=3), ids], lambda b, a: a[0].gather(a[1], "v"))
    assert first.vmap(2, [0, 0]).output_types[0].dims == [("#batch", 2), ("n", 4), ("d", 3)]
    with pytest.raises(T.TensorError) as e:   # 300 rows and one more number do not fit u8
        first.vmap(3, [0, 0])
    assert e.value.name == "UnsupportedBatching"


def test_shard_axes():
    row = [T.spec("f32", n=4, vocab=8), T.spec("i32", n=4)]
    log_prob = T.define("l", row, lambda b, a: a[0].token_log_prob(a[1], "vocab"))
    piece, partial = T.shard_program(log_prob, "n", 2)
    assert not partial and repr(piece.output_types[0]) == "f32[n=2]"
    with pytest.raises(T.SessionError) as e:
        T.shard_program(T.define("l", [T.spec("f32", vocab=8, n=4), row[1]], lambda b, a: a[0].token_log_prob(a[1], "vocab")), "vocab", 2)
    assert "vocabulary" in e.value.message
    look = T.define("g", [T.spec("f32", vocab=8, d=2), T.spec("i32", n=4)], lambda b, a: a[0].gather(a[1], "vocab"))
    assert not T.shard_program(look, "n", 2)[1]
    with pytest.raises(T.SessionError):
        T.shard_program(look, "vocab", 2)
    grad = T.define("s", [T.spec("i32", n=4), T.spec("f32", n=4, d=2)], lambda b, a: nn.embedding_grad(a[0], a[1], "vocab", 8))
    piece, partial = T.shard_program(grad, "n", 2)
    assert partial.name == "sum"
    idx, up = np.array([1, 7, 1, 9], np.int32), np.arange(8, dtype=np.float32).reshape(4, 2)
    parts = [oracle.run(piece.wire, [idx[i:i + 2], up[i:i + 2]])[0] for i in (0, 2)]
    assert np.array_equal(parts[0] + parts[1], oracle.run(grad.wire, [idx, up])[0])
    on_base = T.define("s", [T.spec("f32", vocab=8, d=2), T.spec("i32", n=4), T.spec("f32", n=4, d=2)],
                       lambda b, a: a[0].scatter_add(a[1], a[2], "vocab"))
    with pytest.raises(T.SessionError) as e:
        T.shard_program(on_base, "n", 2)
    assert "base" in e.value.message
    with pytest.raises(T.SessionError):
        T.shard_program(on_base, "vocab", 2)


# ---------------------------------------------------------------------------------------------
# plans
# ---------------------------------------------------------------------------------------------
def plan_lines(session, program):
    compiled = session.compile(program)
    lines = compiled.plan_summary().strip().split("\n")
    session.release(compiled)
    return lines


def test_a_loss_and_its_gradient_read_the_logits_once(cpu_session):
    for program in (policy_program("bf16", batch=4, seq=64, vocab=1000), T.define("ce", [LOGITS, IDS], lambda b, a: nn.cross_entropy(a[0], a[1], "vocab"))):
        lines = plan_lines(cpu_session, program.value_and_grad([0]))
        calls = [x for x in lines if x.startswith("token")]
        assert len(calls) == 1 and "value gradient" in calls[0], lines


def test_a_slope_over_whole_sequences_takes_the_kept_sums(cpu_session):
    def body(b, a):
        per_sequence = a[0].token_log_prob(a[1], "vocab").sum("seq")
        return per_sequence.tanh().sum("batch")
    lines = plan_lines(cpu_session, T.define("seq", [LOGITS, IDS], body).value_and_grad([0]))
    calls = [x for x in lines if x.startswith("token")]
    assert len(calls) == 2 and calls[0].endswith("value") and calls[1].endswith("gradient from kept sums"), lines


def tempered(factor, dtype="bf16"):
    def body(b, a):
        return nn.cross_entropy(a[0].mul(b.scalar(dtype, factor)), a[1], "vocab")
    return body


def test_a_temperature_joins_the_kernel(cpu_session):
    # beyond the factors the kernel takes the product is a kernel of its own; an infinite one is not taken into the gradient either
    for factor, joins, kernels in ((0.5, True, 3), (1024.0, True, 3), (2.0 ** -11, False, 4), (-1.0, False, 4), (float("inf"), False, 5)):
        lines = plan_lines(cpu_session, T.define("t", [LOGITS, IDS], tempered(factor)).value_and_grad([0]))
        calls = [x for x in lines if x.startswith("token")]
        assert len(calls) == 1 and "value gradient" in calls[0], lines
        assert ("scale=%g,%g" % (factor, factor) in calls[0]) == joins and len(lines) == kernels, lines
    # a gradient that something else needs as well is written as it is
    def both(b, a):
        y = a[0].mul(b.scalar("bf16", 0.5))
        return y.token_log_prob(a[1], "vocab").sum(["batch", "seq"]).add(y.token_log_prob(a[2], "vocab").sum(["batch", "seq"]))
    calls = [x for x in plan_lines(cpu_session, T.define("t", [LOGITS, IDS, IDS], both).value_and_grad([0])) if x.startswith("token")]
    assert len(calls) == 2 and all(x.endswith("scale=0.5,1") for x in calls), calls


def test_a_lookup_joins_the_kernel_that_uses_it(cpu_session):
    def norm(b, a):
        x = nn.embedding(a[0], a[1], "vocab", scale=3.0)
        return x.div(x.mul(x).mean("dim").sqrt())
    assert len(plan_lines(cpu_session, T.define("n", [T.spec("f32", vocab=100, dim=64), IDS], norm))) == 1
    # narrow rows: the columns of the kernel do not run over the tokens, whose numbers would then differ per element
    lines = plan_lines(cpu_session, T.define("g", [T.spec("f32", vocab=100, dim=64), T.spec("i32", n=500)], lambda b, a: a[0].gather(a[1], "vocab")))
    assert len(lines) == 1 and "rows=500 cols=64" in lines[0] and "vec=4" in lines[0]


def test_updates_are_computed_where_they_are_summed(cpu_session):
    lines = plan_lines(cpu_session, T.define("s", [T.spec("i32", n=50), T.spec("bf16", n=50, d=8)],
                                             lambda b, a: nn.embedding_grad(a[0], a[1], "vocab", 20, scale=4.0)))
    assert len(lines) == 1 and lines[0].startswith("scatter_add") and "from zeros" in lines[0]


def test_refused_sizes(cpu_session):
    def compile_failed(specs, body, word):
        with pytest.raises(T.SessionError) as e:
            cpu_session.compile(T.define("big", specs, body))
        assert e.value.name == "compile_failed" and word in e.value.message
    compile_failed([T.spec("bf16", n=1, vocab=2 ** 31), T.spec("i32", n=1)], lambda b, a: a[0].token_log_prob(a[1], "vocab"), "not supported")
    compile_failed([T.spec("i64", n=1), T.spec("bf16", n=1)], lambda b, a: nn.embedding_grad(a[0], a[1], "vocab", 2 ** 31), "not supported")


# ---------------------------------------------------------------------------------------------
# on the device
# ---------------------------------------------------------------------------------------------
GATHERS = [  # (data shape, axis, index shape)
    ((11, 8), 0, (5,)), ((1, 1), 0, (1,)), ((300, 1001), 0, (3, 7)), ((7, 64), 0, (1000,)), ((50, 4096), 0, (2, 9)), ((9,), 0, (4, 33)),
    ((6, 13, 10), 1, (4,)), ((5, 3, 17), 2, (2, 6)), ((40, 2, 3), 0, (600,)), ((13, 24), 0, ()), ((2000, 5), 0, (2, 1025)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,axis,index_shape", GATHERS)
@pytest.mark.parametrize("dtype,index", [("f32", "i32"), ("bf16", "i64"), ("f16", "u16"), ("f64", "u32"), ("f32", "i8")])
def test_gather(gpu_session, shape, axis, index_shape, dtype, index):
    rng = np.random.default_rng(len(shape) * 100 + axis)
    specs = [T.spec(dtype, **{"d%d" % i: e for i, e in enumerate(shape)}), T.spec(index, **{"i%d" % i: e for i, e in enumerate(index_shape)})]
    data = stored(dtype, rng.standard_normal(shape))
    low, high = (0 if index[0] == "u" else -2), min(shape[axis] + 2, 120 if index == "i8" else 1 << 14)
    idx = np.asarray(rng.integers(low, high, index_shape)).astype(NP[index])
    want = lookup(exactly(dtype, data), idx, axis)
    plain = T.define("g", specs, lambda b, a: a[0].gather(a[1], "d%d" % axis))
    assert np.array_equal(run(gpu_session, plain, [data, idx])[0], want)
    scaled = T.define("e", specs, lambda b, a: nn.embedding(a[0], a[1], "d%d" % axis, scale=3.0))
    close(run(gpu_session, scaled, [data, idx])[0], 3.0 * want, (U[dtype] + U["f32"] * (dtype != "f64")) * np.abs(3.0 * want) + TINY[dtype])


@pytest.mark.gpu
def test_gather_of_computed_values_and_folds_over_lookups(gpu_session):
    rng = np.random.default_rng(5)
    table, idx, other = rng.standard_normal((37, 48)).astype(np.float32), rng.integers(-1, 38, (6, 70)).astype(np.int32), rng.integers(0, 6, (9,)).astype(np.int32)
    specs = [T.spec("f32", v=37, d=48), T.spec("i32", b=6, n=70), T.spec("i32", m=9)]

    def body(b, a):
        x = a[0].gather(a[1], "v")
        total = x.sum("n")                                            # a fold over the looked-up numbers
        return total, x.mul(x).mean("d"), total.gather(a[2], "b"), a[0].mul(b.scalar("f32", 2.0)).gather(a[1].add(a[1]), "v")
    got = run(gpu_session, T.define("folds", specs, body), [table, idx, other])
    x = lookup(table.astype(np.float64), idx, 0)
    close(got[0], x.sum(1), 72 * U["f32"] * np.abs(x).sum(1))
    close(got[1], (x * x).mean(-1), 52 * U["f32"] * (x * x).mean(-1))
    close(got[2], lookup(x.sum(1), other, 0), 72 * U["f32"] * lookup(np.abs(x).sum(1), other, 0))
    assert np.array_equal(got[3], lookup(2.0 * table.astype(np.float64), idx + idx, 0))


SCATTERS = [  # (base shape, axis, index shape, which indices)
    ((11, 8), 0, (5,), "any"), ((1, 1), 0, (1,), "any"), ((10007, 33), 0, (9, 111), "skewed"), ((50, 4096), 0, (700,), "any"),
    ((300, 24), 0, (4000,), "one"), ((300, 24), 0, (4000,), "none"), ((70000, 8), 0, (5,), "any"), ((40000, 16), 0, (3, 1500), "skewed"),
    ((6, 13, 10), 1, (40,), "any"), ((5, 3, 17), 2, (5, 6), "any"), ((9,), 0, (1000,), "any"), ((13, 24), 0, (), "any"), ((3, 2056), 0, (513,), "any"),
    ((257, 40), 0, (8192,), "sorted"), ((2, 520), 0, (12345,), "skewed"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,axis,index_shape,kind", SCATTERS)
@pytest.mark.parametrize("dtype,index", [("f32", "i32"), ("bf16", "i64"), ("f16", "u32"), ("f64", "i32")])
def test_scatter_add(gpu_session, shape, axis, index_shape, kind, dtype, index):
    rng = np.random.default_rng(shape[0] + axis)
    v = shape[axis]
    idx = np.asarray({"any": lambda: rng.integers(-2 if index[0] == "i" else 0, v + 2, index_shape), "one": lambda: np.full(index_shape, v // 2),
                      "none": lambda: np.full(index_shape, v), "sorted": lambda: np.sort(rng.integers(0, v, index_shape)),
                      "skewed": lambda: (v * rng.random(index_shape) ** 6).astype(np.int64)}[kind]()).astype(NP[index])
    rows = shape[:axis] + tuple(index_shape) + shape[axis + 1:]
    base, up = stored(dtype, rng.standard_normal(shape)), stored(dtype, rng.standard_normal(rows))
    names = ["d%d" % i for i in range(len(shape))]
    inames = ["i%d" % i for i in range(len(index_shape))]
    specs = [T.spec(dtype, **dict(zip(names, shape))), T.spec(index, **dict(zip(inames, index_shape))),
             T.spec(dtype, **dict(zip(names[:axis] + inames + names[axis + 1:], rows)))]
    u = U["f64" if dtype == "f64" else "f32"]
    program = T.define("s", specs, lambda b, a: a[0].scatter_add(a[1], a[2], names[axis]))
    want, mag, n = scattered(exactly(dtype, base), idx, exactly(dtype, up), axis)
    got = run(gpu_session, program, [base, idx, up])[0]
    close(got, want, n * u * mag + U[dtype] * np.abs(want) + TINY[dtype])
    assert np.array_equal(got, run(gpu_session, program, [base, idx, up])[0])
    # from zeros, with the updates computed on the way: 3 * up - up has two roundings of its own
    program = T.define("z", specs[1:], lambda b, a: b.scalar(dtype, 0.0).broadcast(**dict(zip(names, shape))).scatter_add(
        a[0], a[1].mul(b.scalar(dtype, 3.0)).sub(a[1]), names[axis]))
    want, mag, n = scattered(np.zeros(shape), idx, 2.0 * exactly(dtype, up), axis)
    close(run(gpu_session, program, [idx, up])[0], want, (n + 3) * u * mag + U[dtype] * np.abs(want) + TINY[dtype])


@pytest.mark.gpu
def test_scatter_add_of_broadcast_and_transposed_updates(gpu_session):
    rng = np.random.default_rng(8)
    idx = rng.integers(0, 7, (40,)).astype(np.int32)
    specs = [T.spec("f32", v=7, d=12), T.spec("i32", n=40), T.spec("f32", d=12, n=40), T.spec("f32", d=12)]

    def body(b, a):
        ones = b.scalar("f32", 1.0).broadcast(n=40)
        return (a[0].scatter_add(a[1], a[2], "v"), a[0].scatter_add(a[1], a[3], "v"), b.scalar("f32", 0.0).broadcast(v=7).scatter_add(a[1], ones, "v"),
                a[0].scatter_add(a[1], a[2], "v").scatter_add(a[1], a[3], "v"))
    base, up, one = (rng.standard_normal(s).astype(np.float32) for s in ((7, 12), (12, 40), (12,)))
    got = run(gpu_session, T.define("views", specs, body), [base, idx, up, one])
    wide = np.broadcast_to(one.astype(np.float64), (40, 12))
    for g, rows in ((got[0], up.T.astype(np.float64)), (got[1], wide)):
        want, mag, n = scattered(base.astype(np.float64), idx, rows, 0)
        close(g, want, n * U["f32"] * mag + U["f32"] * np.abs(want))
    assert np.array_equal(got[2], np.bincount(idx, minlength=7).astype(np.float64))
    want, mag, n = scattered(base.astype(np.float64), np.concatenate([idx, idx]), np.concatenate([up.T.astype(np.float64), wide]), 0)
    close(got[3], want, (n + 2) * U["f32"] * mag)


ROWS = [((1,), 1), ((1,), 2), ((3,), 7), ((2, 5), 8), ((700,), 9), ((5,), 257), ((3, 3), 1000), ((1,), 4099), ((17,), 33001), ((400,), 5003),
        ((1,), 131072), ((2,), 70001), ((1,), 300007), ((), 50), ((1300,), 64), ((320,), 32768), ((297,), 40003), ((300,), 70001)]


def logits_and_tokens(dtype, rows, vocab, seed, index="i32"):
    rng = np.random.default_rng(seed)
    x = stored(dtype, 3.0 * rng.standard_normal(rows + (vocab,)))
    top = 127 if index == "i8" else 1 << 30
    return x, np.asarray(rng.integers(-1, min(vocab + 1, top), rows)).astype(NP[index])


def axes(rows):
    return {"r%d" % i: e for i, e in enumerate(rows)}


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", ROWS)
@pytest.mark.parametrize("dtype,index", [("f32", "i64"), ("bf16", "i32"), ("f16", "i8")])
def test_token_log_prob_and_its_gradient(gpu_session, rows, vocab, dtype, index):
    x, tok = logits_and_tokens(dtype, rows, vocab, vocab + len(rows), index)
    specs = [T.spec(dtype, **axes(rows), vocab=vocab), T.spec(index, **axes(rows)), T.spec("f32", **axes(rows))]
    xs = exactly(dtype, x)
    want, p, hot, known = log_prob_of(xs, tok)
    allowed = p_error(xs) + 4 * U["f32"] * np.abs(want)
    program = T.define("l", specs[:2], lambda b, a: a[0].token_log_prob(a[1], "vocab"))
    close(run(gpu_session, program, [x, tok])[0], want, allowed)
    if rows == ():
        return
    # a loss whose slope follows from the row's own log-probability, and one that needs all of them first
    weight = np.random.default_rng(3).standard_normal(rows).astype(np.float32)
    weight.reshape(-1)[0] = 0.0
    names = list(axes(rows))
    for sequence in (False, True):
        def body(b, a):
            lp = a[0].token_log_prob(a[1], "vocab").mul(a[2])
            return lp.tanh().sum(names) if not sequence else lp.sum(names).mul(b.scalar("f32", 2.0 ** -10)).tanh()
        value, grad = run(gpu_session, T.define("v", specs, body).value_and_grad([0]), [x, tok, weight])
        wl = weight * want
        t = np.tanh(wl) if not sequence else np.tanh(wl.sum() * 2.0 ** -10)
        slope = weight * (1 - t * t) * (1.0 if not sequence else 2.0 ** -10)
        full = np.where(known, slope, 0.0)[..., None]
        exact = full * (hot - p)
        # the slope: tanh' at a point off by the error of the log-probabilities, and the roundings of 1 - t * t (relative to 1)
        off = (np.abs(weight) * (np.abs(weight) * allowed + 8 * U["f32"]) if not sequence else
               np.abs(weight) * 2.0 ** -10 * ((np.abs(weight) * allowed).sum() * 2.0 ** -10 + (8 + rows[0]) * U["f32"]))
        off = np.where(known, off, 0)[..., None] + 4 * U["f32"] * np.abs(full)
        close(grad, exact, off * (hot + p) + (p_error(xs) + 4 * U["f32"]) * np.abs(full) * (p + hot * U["f32"]) + 4 * U["f32"] * np.abs(full) * hot
              + U[dtype] * np.abs(exact) + TINY[dtype])
        assert np.all(grad[weight == 0] == 0) and np.all(grad[~known] == 0)
        total = t.sum() if not sequence else t
        size = (np.abs(weight) * allowed + 4 * U["f32"] * np.abs(wl)).sum() + (wl.size + 4) * U["f32"] * np.abs(wl).sum()
        close(value.reshape(()), total, size * (1.0 if not sequence else 2.0 ** -10) + 4 * U["f32"] * (1 + np.abs(total)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab,copies", [(9, 1), (1003, 1), (40000, 1), (40001, 34)])
def test_rows_of_infinities_nans_and_lowest_values(gpu_session, dtype, vocab, copies):
    lowest = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": float(synthetic.bf16_bits_to_f32(np.array([0xff7f], np.uint16))[0])}[dtype]
    rng = np.random.default_rng(4)
    x = exactly(dtype, stored(dtype, rng.standard_normal((9, vocab))))
    x[0] = -np.inf                          # nothing left: NaN, as in the formula
    x[1, 3:] = -np.inf                      # three tokens left
    x[2] = lowest                           # all equal: uniform
    x[3, 5:] = lowest                       # five tokens left
    x[4, vocab // 2] = np.inf               # NaN
    x[5, vocab - 1] = np.nan
    x[6] = -lowest
    x[7, 0], x[7, 1:] = -lowest, lowest
    n = 9 * copies   # 306 rows of 40001 pass through shared memory, fewer are held in registers
    x, tok = np.tile(x, (copies, 1)), np.tile(np.array([1, 2, vocab - 1, 1, 0, 0, 3, 0, vocab], np.int32), copies)
    data = stored(dtype, x)
    specs = [T.spec(dtype, n=n, vocab=vocab), T.spec("i32", n=n), T.spec("f32", n=n)]
    want, p, hot, known = log_prob_of(x, tok)
    program = T.define("l", specs, lambda b, a: a[0].token_log_prob(a[1], "vocab").mul(a[2]).sum("n")).grad([0])
    close(run(gpu_session, T.define("l", specs[:2], lambda b, a: a[0].token_log_prob(a[1], "vocab")), [data, tok])[0], want,
          p_error(x) + 4 * U["f32"] * np.abs(np.where(np.isfinite(want), want, 0)))
    g = np.ones(n, np.float32)
    exact = np.where(known[:, None], hot - p, 0)
    with np.errstate(all="ignore"):
        allowed = (p_error(x) + 4 * U["f32"]) * (p + hot) + U[dtype] * np.abs(exact) + TINY[dtype]
    close(run(gpu_session, program, [data, tok, g])[0], exact, allowed)
    # rows whose slope is zero are zero, whatever they hold
    g.reshape(copies, 9)[:, [0, 4, 5]] = 0
    got = run(gpu_session, program, [data, tok, g])[0]
    assert np.all(got.reshape(copies, 9, vocab)[:, [0, 4, 5, 8]] == 0) and np.all(np.isfinite(got))


@pytest.mark.gpu
@pytest.mark.parametrize("factor", [0.5, 3.0, -1.0, 2.0 ** -11, 0.0])
@pytest.mark.parametrize("dtype,rows,vocab", [("f32", 5, 1003), ("bf16", 300, 40000), ("f16", 2, 70001)])
def test_logits_times_a_number(gpu_session, dtype, rows, vocab, factor):
    x, tok = logits_and_tokens(dtype, (rows,), vocab, rows)
    program = T.define("t", [T.spec(dtype, n=rows, vocab=vocab), T.spec("i32", n=rows)], tempered(factor, dtype)).value_and_grad([0])
    value, grad = run(gpu_session, program, [x, tok])
    y = factor * exactly(dtype, x)
    want, p, hot, known = log_prob_of(y, tok)
    n = max(known.sum(), 1)
    step = p_error(y) + 2 * U["f32"] * (1 + spread_of(y))   # the product is rounded, or the constant that takes its place
    close(value.reshape(()), -want.sum() / n, step + (rows + 8) * U["f32"] * np.abs(want).sum() / n)
    exact = factor * (p - hot) * known[:, None] / n
    close(grad, exact, abs(factor) / n * known[:, None] * (p + hot) * (step + 8 * U["f32"]) + U[dtype] * np.abs(exact) + TINY[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["gather", "scatter_add", "log_prob"])
def test_batched_and_forward_mode_programs_on_the_device(gpu_session, op):
    """vmap with both operands mapped, and jvp, against the oracle's f64 evaluation of the same derived programs: short f32
    sums, 40 roundings of the largest magnitude at most."""
    rng = np.random.default_rng(2)
    v, n, d, size = 70, 48, 48, 5

    def body(b, a):
        if op == "gather":
            return a[0].gather(a[1], "v")
        if op == "scatter_add":
            return a[0].scatter_add(a[1], a[0].gather(a[1], "v").mul(b.scalar("f32", 2.0)), "v")
        return a[0].token_log_prob(a[1].rename("n", "d"), "v")
    program = T.define("one", [T.spec("f32", v=v, d=d), T.spec("i32", n=n)], body)
    x, idx = rng.standard_normal((size, v, d)).astype(np.float32), rng.integers(-2, v + 2, (size, n)).astype(np.int32)
    for derived, inputs in ((program.vmap(size, [0, 0]), [x, idx]), (program.jvp([0]), [x[0], idx[0], x[1]]),
                            (program.jvp([0]).vmap(size, [0, 0, None]), [x, idx, x[1]])):
        for got, want in zip(run(gpu_session, derived, inputs), oracle.run(derived.wire, inputs, mode="f64")):
            close(got, want, 40 * U["f32"] * (np.abs(want) + np.abs(want).max()) + p_error(x.astype(np.float64)) * np.abs(want).max())


@pytest.mark.gpu
def test_policy_gradients_of_every_input_on_the_device(gpu_session):
    inputs = policy_case("f32", 3, 70, 1003, 5)
    program = policy_program("f32", "i32", 3, 70, 1003).value_and_grad([0, 2, 3, 4])
    for got, want in zip(run(gpu_session, program, inputs), oracle.run(program.wire, inputs, mode="f64")):
        # ratios off by the error of a log-probability, then f32 sums of at most 210 terms
        scale = np.abs(want).max()
        close(got.reshape(want.shape), want, (4 * p_error(exactly("f32", inputs[0])) + 300 * U["f32"]) * (np.abs(want) + scale))


@pytest.mark.gpu
def test_the_vocabulary_may_be_any_axis(gpu_session):
    rng = np.random.default_rng(9)
    x, tok = rng.standard_normal((5, 40, 6)).astype(np.float32), rng.integers(-1, 40, (6, 5)).astype(np.int32)
    program = T.define("m", [T.spec("f32", a=5, vocab=40, c=6), T.spec("i32", c=6, a=5)], lambda b, a: nn.cross_entropy(a[0], a[1], "vocab")).value_and_grad([0])
    value, grad = run(gpu_session, program, [x, tok])
    want, p, hot, known = log_prob_of(np.moveaxis(x, 1, 2).astype(np.float64), tok.T)
    n = max(known.sum(), 1)
    close(value.reshape(()), -want.sum() / n, 1e-6)
    close(grad, np.moveaxis((p - hot) * known[..., None] / n, 2, 1), 1e-7)


def policy_case(dtype, batch, seq, vocab, seed, index="i32"):
    x, tok = logits_and_tokens(dtype, (batch, seq), vocab, seed, index)
    rng = np.random.default_rng(seed + 1)
    now = log_prob_of(exactly(dtype, x), tok)[0]
    off = 0.15 * rng.standard_normal((batch, seq))
    # no ratio within a hundredth of a border, where one rounding decides about a row
    off[np.abs(np.exp(off) - 0.8) < 0.01] = 0
    off[np.abs(np.exp(off) - 1.2) < 0.01] = 0
    mask = (np.arange(seq) < rng.integers(0, seq + 1, (batch, 1))).astype(np.float32)
    return [x, tok, (now - off).astype(np.float32), (now + 0.3 * rng.standard_normal((batch, seq))).astype(np.float32),
            rng.standard_normal(batch).astype(np.float32), mask]


def policy_exact(dtype, x, tok, old, reference, advantage, mask, clip=0.2, kl=0.05):
    """(loss, gradient, slope, what the slope may be off by) in f64"""
    xs = exactly(dtype, x)
    log_p, p, hot, known = log_prob_of(xs, tok)
    weight = np.where(known & (mask != 0), mask, 0).astype(np.float64)
    on = weight != 0
    log_p, old, reference = (np.where(on, v, 0).astype(np.float64) for v in (log_p, old, reference))
    a = advantage.astype(np.float64)[:, None]
    r, d, n = np.exp(log_p - old), reference - log_p, max(weight.sum(), 1)
    free, held = r * a, np.clip(r, 1 - clip, 1 + clip) * a
    loss = (weight * (kl * (np.exp(d) - d - 1) - np.minimum(free, held))).sum() / n
    slope = weight / n * (kl * (1 - np.exp(d)) - np.where(free <= held, free, 0))
    step = p_error(xs) + 16 * U["f32"] * (1 + np.abs(log_p))
    off = weight / n * (kl * (np.exp(d) + 1) + np.abs(free)) * step + 4 * U["f32"] * np.abs(slope)
    g = slope[..., None]
    grad = np.where(g == 0, 0, g * (hot - np.where(g == 0, 0, p)))
    bound = off[..., None] * (hot + np.where(g == 0, 0, p)) + (p_error(xs) + 8 * U["f32"]) * np.abs(g) * np.where(g == 0, 0, p + hot) + U[dtype] * np.abs(grad) + TINY[dtype]
    # the loss: each term's error, and a sum of batch * seq terms
    each = weight / n * (kl * (np.exp(d) + np.abs(d) + 1) + np.abs(free))
    return loss, grad, bound, (each * step).sum() + (weight.size + 8) * U["f32"] * each.sum()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,seq,vocab", [(1, 1, 3), (2, 3, 11), (4, 65, 1000), (3, 100, 33003), (2, 2, 140001), (9, 130, 64)])
@pytest.mark.parametrize("dtype,index", [("f32", "i64"), ("bf16", "i32"), ("f16", "i32")])
def test_policy_loss_and_gradient(gpu_session, batch, seq, vocab, dtype, index):
    inputs = policy_case(dtype, batch, seq, vocab, vocab + batch, index)
    value, grad = run(gpu_session, policy_program(dtype, index, batch, seq, vocab).value_and_grad([0]), inputs)
    loss, exact, bound, loss_bound = policy_exact(dtype, *inputs)
    close(value.reshape(()), loss, loss_bound)
    close(grad, exact, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("loss", ["policy", "cross_entropy"])
def test_nothing_at_a_masked_position_reaches_a_loss(gpu_session, loss):
    inputs = policy_case("bf16", 4, 40, 515, 77)
    mask = inputs[5]
    mask[:] = 1
    mask[1] = 0
    mask[2, 7:] = 0
    off = mask == 0
    if loss == "policy":
        program, use = policy_program("bf16", batch=4, seq=40, vocab=515).value_and_grad([0]), lambda i: i
    else:
        program = T.define("ce", [T.spec("bf16", batch=4, seq=40, vocab=515), T.spec("i32", batch=4, seq=40), T.spec("f32", batch=4, seq=40)],
                           lambda b, a: nn.cross_entropy(a[0], a[1], "vocab", mask=a[2])).value_and_grad([0])
        use = lambda i: [i[0], i[1], i[5]]  # noqa: E731
    clean = run(gpu_session, program, use(inputs))
    dirty = [x.copy() for x in inputs]
    dirty[0][off] = 0x7fc0                     # NaN
    dirty[1][off] = np.iinfo(np.int32).min
    dirty[2][off], dirty[3][off] = np.nan, np.inf
    dirty[4][1] = np.inf                       # the advantage of the sequence that is masked altogether
    got = run(gpu_session, program, use(dirty))
    assert np.array_equal(got[0], clean[0]) and np.array_equal(got[1], clean[1]) and np.all(np.isfinite(clean[1]))
    assert np.all(got[1][off] == 0)
    # tokens outside the vocabulary count like masked ones; nothing left gives zero
    dirty[1][:] = -1
    got = run(gpu_session, program, use(dirty))
    assert float(got[0].reshape(-1)[0]) == 0 and np.all(got[1] == 0)


@pytest.mark.gpu
def test_empty_axes(gpu_session):
    table, none = np.ones((4, 3), np.float32), np.zeros((0,), np.int32)
    p = T.define("g", [T.spec("f32", v=4, d=3), T.spec("i32", n=0)], lambda b, a: (a[0].gather(a[1], "v").sum("n"), a[0].scatter_add(a[1], a[0].gather(a[1], "v"), "v")))
    got = run(gpu_session, p, [table, none])
    assert np.array_equal(got[0], np.zeros(3)) and np.array_equal(got[1], table)
    p = T.define("g", [T.spec("f32", v=0, d=3), T.spec("i32", n=5)], lambda b, a: a[0].gather(a[1], "v"))
    assert np.array_equal(run(gpu_session, p, [np.zeros((0, 3), np.float32), np.zeros(5, np.int32)])[0], np.zeros((5, 3)))
    p = T.define("l", [T.spec("f32", n=5, v=0), T.spec("i32", n=5)], lambda b, a: a[0].token_log_prob(a[1], "v"))
    assert np.array_equal(run(gpu_session, p, [np.zeros((5, 0), np.float32), np.zeros(5, np.int32)])[0], np.zeros(5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", [(2, 3, 11, 6), (4, 64, 1000, 128), (2, 33, 257, 72)])
def test_lookup_head_loss_and_both_gradients_together(gpu_session, dtype, sizes):
    """A whole step on the token side: lookup, a nonlinearity, logits against the same table, the loss, and the
    table's gradient, which joins a contraction and a scatter.  Against the f64 evaluation of the same program by the oracle."""
    batch, seq, vocab, dim = sizes
    inputs = head_inputs(batch, seq, vocab, dim)
    inputs[0] = stored(dtype, inputs[0])
    program = head_program(dtype, batch, seq, vocab, dim).value_and_grad([0])
    got = run(gpu_session, program, inputs)
    want = oracle.run(program.wire, inputs, mode="f64")
    # 16-bit values are rounded where a contraction reads them (hidden state, gradient of the logits) and at the end:
    # three roundings on the way to each gradient; f32 sums of up to vocab + batch * seq terms otherwise
    scale = np.abs(want[1]).max()
    close(got[1], want[1], 4 * U[dtype] * (np.abs(want[1]) + scale) + 1e-5 * scale)
    close(got[0].reshape(()), want[0].reshape(()), (4 * U[dtype] + 1e-5) * abs(float(want[0].reshape(-1)[0])))


def random_token_program(seed):
    """A lookup in a table of one to three axes by numbers of none to two, what follows it elementwise, folds of it, a scatter back
    into the table, a second lookup and the log-probability of tokens along some axis of it, with a gradient."""
    rng = np.random.default_rng(900 + seed)
    pick = lambda *xs: xs[rng.integers(len(xs))]  # noqa: E731
    extent = lambda: int(pick(1, 2, 3, 5, 8, 16, 33, 64, 130))  # noqa: E731
    table = {"t%d" % i: extent() for i in range(rng.integers(1, 4))}
    axis = pick(*table)
    ids = {"i%d" % i: extent() for i in range(rng.integers(0, 3))}
    looked = [n for n in list(table)[:list(table).index(axis)]] + list(ids) + [n for n in list(table)[list(table).index(axis) + 1:]]
    dims = {**table, **ids}
    specs = [T.spec("f32", **table), T.spec(pick("i32", "i64", "i16"), **ids)]
    bias = {n: dims[n] for n in looked if rng.random() < 0.5}
    specs.append(T.spec("f32", **dict(reversed(list(bias.items())))))
    vocab = pick(*looked) if looked else None
    if vocab:
        specs.append(T.spec("i32", **{n: dims[n] for n in reversed(looked) if n != vocab}))
    transposed, fold = rng.random() < 0.4, pick(*looked) if looked else None

    def body(b, a):
        source = a[0].mul(b.scalar("f32", 1.5)) if transposed else a[0]
        x = source.gather(a[1], axis)
        y = x.mul(x).sub(a[2])
        outs = [y, a[0].scatter_add(a[1], y.mul(b.scalar("f32", 0.5)), axis)]
        if fold:
            outs += [y.sum(fold), x.max(fold)]
        if vocab:
            outs.append(y.token_log_prob(a[3], vocab))
        return outs

    def loss(b, a):
        x = a[0].gather(a[1], axis)
        y = x.mul(a[2]).add(x)
        total = y.sum(list(looked)) if looked else y
        if vocab:
            log_prob = y.token_log_prob(a[3], vocab)
            names = [n for n, _ in log_prob.ty.dims]
            total = total.add(log_prob.sum(names) if names else log_prob)
        return total
    inputs = []
    for s in specs:
        shape = tuple(e for _, e in s.dims)
        if s.dtype == "f32":
            inputs.append(rng.standard_normal(shape).astype(np.float32))
        else:
            top = table[axis] if len(inputs) == 1 else dims[vocab]
            inputs.append(np.asarray(rng.integers(-1, top + 1, shape)).astype(NP[s.dtype]))
    return specs, body, loss, inputs


@pytest.mark.parametrize("seed", range(32))
def test_random_token_programs_plan(cpu_session, seed):
    specs, body, loss, _ = random_token_program(seed)
    for program in (T.define("r", specs, body), T.define("l", specs, loss).value_and_grad([0, 2])):
        compiled = cpu_session.compile(program)
        cpu_session.release(compiled)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(32))
def test_random_token_programs_match_the_oracle(gpu_session, seed):
    """Values of size about one, f32 sums of at most 130 * 130 of them and exponentials of them: 1e-5 of the largest
    magnitude (sums of n terms of both signs: n * 2^-24 * mean magnitude at most, reached by no fold in trees).  The gradient
    at a token is g - g * p: four roundings of g, which is 1 here, also where p is 1 and nothing else is left (a vocabulary of
    one), times the derivative 1 + bias of y, at most 6 in these inputs: 6 * 4 * 2^-24 < 2e-6."""
    specs, body, loss, inputs = random_token_program(seed)
    for program in (T.define("r", specs, body), T.define("l", specs, loss).value_and_grad([0, 2])):
        for got, want in zip(run(gpu_session, program, inputs), oracle.run(program.wire, inputs, mode="f64")):
            want = np.asarray(want).reshape(got.shape)
            close(got, want, 1e-5 * (np.abs(want) + (np.abs(want).max() if want.size else 0)) + 2e-6)


def torch_buffers(program, inputs):
    import torch
    given = [torch.from_numpy(np.ascontiguousarray(x.view(np.int16) if x.dtype == np.uint16 else x)).cuda() for x in inputs]
    kinds = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
    return given, [torch.full(shape_of(t), 5.0, dtype=kinds[t.dtype], device="cuda") for t in program.output_types]


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["policy", "embedding_grad", "embedding", "log_prob"])
def test_captured_replayed_and_on_other_streams(which):
    """Device buffers on the default stream, on a side stream and captured into a CUDA graph: the replays follow the inputs."""
    import torch
    cases = []
    for seed in (1, 2):
        rng = np.random.default_rng(seed)
        ids = rng.integers(-1, 300, (4, 65)).astype(np.int32)
        if which == "policy":
            cases.append(policy_case("bf16", 4, 65, 1003, seed))
        elif which == "embedding_grad":
            cases.append([ids, rng.standard_normal((4, 65, 72)).astype(np.float32)])
        elif which == "embedding":
            cases.append([rng.standard_normal((300, 72)).astype(np.float32), ids])
        else:
            cases.append([rng.standard_normal((4, 65, 300)).astype(np.float32), ids])
    if which == "policy":
        program = policy_program("bf16", "i32", 4, 65, 1003).value_and_grad([0])
    elif which == "embedding_grad":
        program = T.define("s", [T.spec("i32", b=4, n=65), T.spec("f32", b=4, n=65, d=72)], lambda b, a: nn.embedding_grad(a[0], a[1], "v", 300, scale=2.0))
    elif which == "embedding":
        program = T.define("e", [T.spec("f32", v=300, d=72), T.spec("i32", b=4, n=65)], lambda b, a: nn.embedding(a[0], a[1], "v", scale=2.0))
    else:
        program = T.define("l", [T.spec("f32", b=4, n=65, v=300), T.spec("i32", b=4, n=65)], lambda b, a: a[0].token_log_prob(a[1], "v"))
    cuda = T.Cuda(program, device=0)
    want = []
    for inputs in cases:
        outs = [np.zeros(shape_of(t), NP[t.dtype]) for t in program.output_types]
        cuda.launch(inputs, outs)
        want.append([exactly(t.dtype, o) for t, o in zip(program.output_types, outs)])
    given, outs = torch_buffers(program, cases[0])
    later = torch_buffers(program, cases[1])[0]

    def fresh():
        for o in outs:
            o.fill_(7.0)

    def same(k):
        torch.cuda.synchronize()
        return all(np.array_equal(o.double().cpu().numpy(), w.reshape(shape_of(t))) for o, w, t in zip(outs, want[k], program.output_types))

    def launch(stream):
        cuda.launch_device([x.data_ptr() for x in given], [x.data_ptr() for x in outs], stream)
    for _ in range(3):   # the legacy default stream
        fresh()
        launch(1)
        assert same(0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    fresh()
    torch.cuda.synchronize()
    launch(side.cuda_stream)
    assert same(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        launch(side.cuda_stream)
    for k in (0, 1, 0):
        for x, y, z in zip(given, later, torch_buffers(program, cases[0])[0]):
            x.copy_(y if k else z)
        fresh()
        torch.cuda.synchronize()
        graph.replay()
        assert same(k)
    fresh()
    torch.cuda.synchronize()
    launch(side.cuda_stream)   # an ordinary call after the replays
    assert same(0)
    del graph
    cuda.deinit()


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Buffers of more than 2^32 bytes and 2^31 elements: the rows at both ends of a table, of its gradient, and of a batch of logits."""
    import torch
    free = torch.cuda.mem_get_info()[0]
    if free < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    vocab, dim = 600011, 4096
    table = torch.zeros(vocab, dim, dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([0, vocab - 1, 524287, 524288, vocab - 1, -1, vocab], dtype=torch.int64, device="cuda")
    known = ids.clamp(0, vocab - 1)
    table[known] = torch.randn(7, dim, device="cuda").bfloat16()
    torch.cuda.synchronize()
    rows = torch.full((7, dim), 3.0, dtype=torch.bfloat16, device="cuda")
    program = T.define("e", [T.spec("bf16", v=vocab, d=dim), T.spec("i64", n=7)], lambda b, a: nn.embedding(a[0], a[1], "v", scale=2.0))
    cuda = T.Cuda(program, device=0)
    cuda.launch_device([table.data_ptr(), ids.data_ptr()], [rows.data_ptr()], 1)
    torch.cuda.synchronize()
    want = table[known] * 2.0
    want[5:] = 0
    assert torch.equal(rows, want)
    cuda.deinit()
    # the gradient over the same table: row sums at both ends, zeros elsewhere
    up = torch.randn(7, dim, device="cuda").bfloat16()
    out = table
    out.fill_(9.0)
    program = T.define("s", [T.spec("i64", n=7), T.spec("bf16", n=7, d=dim)], lambda b, a: nn.embedding_grad(a[0], a[1], "v", vocab))
    cuda = T.Cuda(program, device=0)
    cuda.launch_device([ids.data_ptr(), up.data_ptr()], [out.data_ptr()], 1)
    torch.cuda.synchronize()
    expected = {0: up[0], vocab - 1: (up[1].float() + up[4].float()).bfloat16(), 524287: up[2], 524288: up[3]}
    for row, values in expected.items():
        assert torch.equal(out[row], values)
    out[list(expected)] = 0
    assert not bool(out.any())
    cuda.deinit()
    del table, out
    # logits of 36007 x 60001: the last rows start beyond 2^32 bytes
    n, v = 36007, 60001
    logits = torch.zeros(n, v, dtype=torch.bfloat16, device="cuda")
    tok = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    at = [0, 35789, 35794, n - 1]     # 35794 * 60001 is the first element past 2^31
    logits[at] = torch.randn(4, v, device="cuda").bfloat16()
    tok[at] = torch.tensor([5, 0, 60000, 31], dtype=torch.int32, device="cuda")
    loss, grad = torch.zeros((), device="cuda"), torch.full((n, v), 7.0, dtype=torch.bfloat16, device="cuda")
    program = T.define("c", [T.spec("bf16", n=n, v=v), T.spec("i32", n=n)], lambda b, a: nn.cross_entropy(a[0], a[1], "v")).value_and_grad([0])
    cuda = T.Cuda(program, device=0)
    torch.cuda.synchronize()
    cuda.launch_device([logits.data_ptr(), tok.data_ptr()], [loss.data_ptr(), grad.data_ptr()], 1)
    torch.cuda.synchronize()
    x, t = logits[at].double().cpu().numpy(), tok[at].cpu().numpy()
    log_p, p, hot, _ = log_prob_of(x, t)
    close(float(loss), -log_p.sum() / 4, p_error(x) + 8 * U["f32"] * 12)
    exact = (p - hot) / 4
    close(grad[at].double().cpu().numpy(), exact, (p_error(x) + 8 * U["f32"]) * (p + hot) / 4 + U["bf16"] * np.abs(exact) + TINY["bf16"])
    grad[at] = 0
    assert not bool(grad.any())
    cuda.deinit()


@pytest.mark.gpu
def test_host_invoke_in_chunks_equals_one_shot():
    """A large lookup and a large scoring call stream through the device in chunks; the table's gradient does not."""
    rng = np.random.default_rng(6)
    table, ids = rng.standard_normal((5000, 1024)).astype(np.float32), rng.integers(-1, 5000, (64, 512)).astype(np.int32)
    logits, tok = rng.standard_normal((64, 128, 2500)).astype(np.float32), rng.integers(0, 2500, (64, 128)).astype(np.int32)
    programs = [(T.define("e", [T.spec("f32", v=5000, d=1024), T.spec("i32", b=64, n=512)], lambda b, a: nn.embedding(a[0], a[1], "v", scale=2.0)), [table, ids]),
                (T.define("l", [T.spec("f32", b=64, n=128, v=2500), T.spec("i32", b=64, n=128)], lambda b, a: a[0].token_log_prob(a[1], "v")), [logits, tok])]
    for program, inputs in programs:
        results = []
        for single in (0, 1):
            session = T.Session(device=0, single_shot_invoke=single)
            results.append(run(session, program, inputs)[0])
            session.deinit()
        assert np.array_equal(results[0], results[1])
