"""Losses on token log-probabilities in the company they keep: logits times a number (a temperature) that something else
reads too, slopes over whole sequences, several log-probabilities in one loss.

CPU: what the planner makes of them.  GPU: values and gradients against the oracle's f64 evaluation of the same programs.
"""
import numpy as np
import pytest

from accy_b200 import tensor
from oracle import oracle
from test_token_programs import close, exactly, p_error, plan_lines, run, stored, U

T = tensor


def token_calls(lines):
    """(line, factor on the logits) of every token kernel of a plan"""
    calls = [x for x in lines if x.startswith("token log-probabilities")]
    return [(x, float(x.split("scale=")[1].split(",")[0]) if "scale=" in x else 1.0) for x in calls]


# ---------------------------------------------------------------------------------------------
# sums kept for a gradient belong to the logits, and the factor, they were made from
# ---------------------------------------------------------------------------------------------
def whole_sequence(factor, dtype, company):
    """tanh of the log-probability of a whole sequence under logits times a number; where a contraction of the product is a
    second factor of the loss, the log-probability's slope needs the product in a buffer."""
    def body(b, a):
        y = a[0].mul(b.scalar(dtype, factor))
        n = dict(a[1].ty.dims)["n"]
        likely = lambda: y.token_log_prob(a[1], "vocab").sum("n").mul(b.scalar("f32", 1.0 / (64 * n))).tanh()  # noqa: E731
        if company == "alone":
            return likely()
        if company == "contraction first":
            return y.contract(a[2], "vocab").sum(["n", "d"]).mul(likely())
        return likely().mul(y.contract(a[2], "vocab").sum(["n", "d"]))
    return body


def whole_sequence_program(company, factor, dtype="f32", n=6, vocab=40, d=5):
    specs = [T.spec(dtype, n=n, vocab=vocab), T.spec("i32", n=n), T.spec(dtype, vocab=vocab, d=d)]
    return T.define("sequence", specs, whole_sequence(factor, dtype, company)).value_and_grad([0])


@pytest.mark.parametrize("factor", [0.5, 2.0, 30.0])
@pytest.mark.parametrize("company", ["alone", "contraction first", "contraction last"])
def test_value_and_gradient_of_a_sequence_read_the_same_logits(cpu_session, company, factor):
    calls = token_calls(plan_lines(cpu_session, whole_sequence_program(company, factor)))
    assert len(calls) == 2 and "from kept sums" in calls[1][0]
    assert calls[0][1] == calls[1][1], calls


@pytest.mark.gpu
@pytest.mark.parametrize("factor", [0.5, 2.0, 30.0])
@pytest.mark.parametrize("company,dtype", [("alone", "f32"), ("alone", "bf16"), ("contraction first", "f32"), ("contraction last", "f32")])
@pytest.mark.parametrize("vocab", [40, 5003])
def test_gradients_of_sequences_under_a_temperature(gpu_session, company, dtype, factor, vocab):
    """f32 throughout: sums of at most 7 * vocab terms (the contraction's), a product rounded at its size, and the error of a
    probability, each relative to the magnitude of what is summed: the contraction C (|C| <= size, its own gradient is a
    row of w summed over d), and a log-probability's slope, 1 / (64 n) at most."""
    rng = np.random.default_rng(vocab)
    n, d = 7, 5
    x, w = stored(dtype, rng.standard_normal((n, vocab))), stored(dtype, rng.standard_normal((vocab, d)) / np.sqrt(vocab))
    tok = rng.integers(-1, vocab + 1, (n,)).astype(np.int32)
    program = whole_sequence_program(company, factor, dtype, n, vocab, d)
    got, want = run(gpu_session, program, [x, tok, w]), oracle.run(program.wire, [x, tok, w], mode="f64")
    y, ws = factor * exactly(dtype, x), np.abs(exactly(dtype, w))
    step = p_error(y) + 4 * U["f32"] * (1 + np.abs(y).max()) + 7 * vocab * U["f32"]
    size, row = (1.0, 0.0) if company == "alone" else (float((np.abs(y) @ ws).sum()), float(ws.sum(1).max()))
    grad = want[1].reshape(got[1].shape)
    close(got[1], grad, 2 * step * factor * (size / (64 * n) + row) + U[dtype] * np.abs(grad))
    close(got[0].reshape(()), float(want[0].reshape(-1)[0]), 2 * step * size)
