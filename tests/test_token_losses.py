"""Losses on token log-probabilities in the company they keep: logits times a number (a temperature) that something else
reads too, slopes over whole sequences, several log-probabilities in one loss.

CPU: what the planner makes of them.  GPU: values and gradients against the oracle's f64 evaluation of the same programs.
"""
import numpy as np
import pytest

from accy_b200 import nn, tensor
from oracle import oracle
from test_token_programs import TINY, U, close, exactly, log_prob_of, p_error, plan_lines, run, stored

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


# ---------------------------------------------------------------------------------------------
# a gradient whose product with a number is one value among others of a region
# ---------------------------------------------------------------------------------------------
def scaled(b, x, factor):
    return x.mul(b.scalar(x.ty.dtype, factor))


def soft_capped(b, x):
    return scaled(b, scaled(b, x, 1.0 / 32).tanh(), 32.0)


def beside(name):
    """(body, names of the inputs, which of them are differentiated) of a loss on scaled logits beside something else"""
    tokens = lambda b, x, a: nn.cross_entropy(x, a["tok"], "vocab")  # noqa: E731
    return {
        "soft cap": (lambda b, a: tokens(b, soft_capped(b, a["x"]), a), ["x", "tok"], [0]),
        "soft cap of a contraction": (lambda b, a: tokens(b, soft_capped(b, a["h"].contract(a["w"], "d")), a), ["h", "w", "tok"], [0, 1]),
        "scaled and plain": (lambda b, a: tokens(b, scaled(b, a["x"], 0.5), a).add(tokens(b, a["x"], a)), ["x", "tok"], [0]),
        "two temperatures": (lambda b, a: tokens(b, scaled(b, a["x"], 0.5), a).add(tokens(b, scaled(b, a["x"], 2.0), a)), ["x", "tok"], [0]),
        "a bias alone": (lambda b, a: tokens(b, scaled(b, a["x"].add(a["bias"]), 0.5), a), ["x", "tok", "bias"], [2]),
        "centred": (lambda b, a: tokens(b, scaled(b, a["x"].sub(a["x"].mean("vocab")), 0.5), a), ["x", "tok"], [0]),
        "squares": (lambda b, a: tokens(b, scaled(b, a["x"], 0.5), a).add(scaled(b, a["x"].mul(a["x"]).sum(["n", "vocab"]), 2.0 ** -10)), ["x", "tok"], [0]),
        "squares and a sequence": (lambda b, a: scaled(b, scaled(b, a["x"], 0.5).token_log_prob(a["tok"], "vocab").sum("n"), 1.0 / 64).tanh().add(
            scaled(b, a["x"].mul(a["x"]).sum(["n", "vocab"]), 2.0 ** -10)), ["x", "tok"], [0]),
        "the same twice": (lambda b, a: tokens(b, scaled(b, a["x"], 0.5), a).add(tokens(b, scaled(b, a["x"], 0.5), a)), ["x", "tok"], [0]),
        "the same under another number": (lambda b, a: tokens(b, scaled(b, a["x"], 0.5), a).add(scaled(b, tokens(b, scaled(b, a["x"], 0.5), a), 3.0)), ["x", "tok"], [0]),
    }[name]


BESIDE = [(name, dtype) for name in ("soft cap", "soft cap of a contraction", "scaled and plain", "two temperatures", "a bias alone", "centred",
                                     "squares", "squares and a sequence", "the same twice", "the same under another number")
          for dtype in ("f32", "bf16") if dtype == "f32" or "squares" not in name]   # a sum of bf16 squares is no f32 term of a loss


def beside_program(name, dtype, n=6, vocab=40, d=8):
    body, names, wrt = beside(name)
    specs = {"x": T.spec(dtype, n=n, vocab=vocab), "tok": T.spec("i32", n=n), "bias": T.spec(dtype, vocab=vocab), "h": T.spec(dtype, n=n, d=d), "w": T.spec(dtype, d=d, vocab=vocab)}
    return T.define("beside", [specs[k] for k in names], lambda b, a: body(b, dict(zip(names, a)))), names, wrt


@pytest.mark.parametrize("name,dtype", BESIDE)
def test_losses_on_scaled_logits_beside_other_things_plan(cpu_session, name, dtype):
    program, _, wrt = beside_program(name, dtype)
    for derived in (program.value_and_grad(wrt), program.grad(wrt)):
        assert token_calls(plan_lines(cpu_session, derived))


def beside_magnitudes(name, wrt, inputs, n):
    """(largest |gradient| the terms of each differentiated input can add up to, |value| its terms can), from
    |d log p / d logit| <= 1, |tanh'| <= 1 and the numbers of the program"""
    x = np.abs(inputs["x"]).max()
    per_logit = {"scaled and plain": 1.5 / n, "two temperatures": 2.5 / n, "centred": 2 * 0.5 / n, "a bias alone": 0.5, "squares": 0.5 / n + 2.0 ** -9 * x,
                 "squares and a sequence": 0.5 / 64 + 2.0 ** -9 * x, "the same twice": 1.0 / n, "the same under another number": 2.0 / n}.get(name, 1.0 / n)
    squares = 2.0 ** -10 * (inputs["x"] ** 2).sum() if "squares" in name else 0.0
    if name == "soft cap of a contraction":   # sum_v |d / d logit| <= 2 / n per row
        return [2.0 / n * np.abs(inputs["w"]).max(), np.abs(inputs["h"]).max()], 1.0
    return [per_logit] * len(wrt), 1.0 + squares


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [(6, 40, 8), (310, 5003, 64), (299, 33001, 8)])
@pytest.mark.parametrize("name,dtype", BESIDE)
def test_losses_on_scaled_logits_beside_other_things(gpu_session, name, dtype, sizes):
    """Elementwise operations round at the size of their results (tanh to two roundings), sums have at most n, vocab or n * vocab
    terms; a contraction reads the 16-bit rounding of the logits' gradient and sums f32 products."""
    n, vocab, d = sizes
    rng = np.random.default_rng(n)
    program, names, wrt = beside_program(name, dtype, n, vocab, d)
    values = {"x": stored(dtype, 2.0 * rng.standard_normal((n, vocab))), "tok": rng.integers(-1, vocab + 1, (n,)).astype(np.int32),
              "bias": stored(dtype, rng.standard_normal(vocab)), "h": stored(dtype, rng.standard_normal((n, d))),
              "w": stored(dtype, rng.standard_normal((d, vocab)))}
    inputs = [values[k] for k in names]
    derived = program.value_and_grad(wrt)
    got, want = run(gpu_session, derived, inputs), oracle.run(derived.wire, inputs, mode="f64")
    exact = {k: exactly(dtype, v) if k != "tok" else v for k, v in values.items()}
    logits = exact["h"] @ exact["w"] if "contraction" in name else exact["x"] + (exact["bias"] if "bias" in name else 0)
    top = np.abs(logits).max() * (2.0 if name == "two temperatures" else 1.0)
    sums = (n + vocab + 64) * U["f32"]
    # what a logit is off by moves a probability by as much, relative to it
    step = p_error(2.0 * logits) + 16 * U["f32"] * (1 + top) + (d * U["f32"] * (np.abs(exact["h"]) @ np.abs(exact["w"])).max() if "contraction" in name else 0)
    magnitudes, size = beside_magnitudes(name, wrt, exact, n)
    close(got[0].reshape(()), float(want[0].reshape(-1)[0]), (2 * step + sums) * (size + np.abs(float(want[0].reshape(-1)[0]))))
    for g, w, m in zip(got[1:], want[1:], magnitudes):
        w = w.reshape(g.shape)
        close(g, w, (2 * step + sums + (U[dtype] if "contraction" in name else 0)) * m + U[dtype] * np.abs(w))


# ---------------------------------------------------------------------------------------------
# log-probabilities that are each other's slopes
# ---------------------------------------------------------------------------------------------
def entangled(name):
    """(body of (logits, tokens, other logits, other tokens), which inputs are differentiated)"""
    mean = lambda b, x: x.sum(["s", "n"]).mul(b.scalar("f32", 1.0 / 16))  # noqa: E731
    lp = lambda a, i, j: a[i].token_log_prob(a[j], "vocab")  # noqa: E731
    return {
        "weight": (lambda b, a: mean(b, lp(a, 0, 1).mul(lp(a, 2, 3).exp())), [0, 2]),
        "product of losses": (lambda b, a: nn.cross_entropy(a[0], a[1], "vocab").mul(nn.cross_entropy(a[2], a[3], "vocab")), [0, 2]),
        "product of sequences": (lambda b, a: lp(a, 0, 1).sum("n").mul(lp(a, 2, 3).sum("n")).sum("s").mul(b.scalar("f32", 1.0 / 256)), [0, 2]),
        "preference": (lambda b, a: lp(a, 0, 1).sum("n").sub(lp(a, 2, 3).sum("n")).mul(b.scalar("f32", 1.0 / 32)).tanh().sum("s"), [0, 2]),
        "two token sets": (lambda b, a: mean(b, lp(a, 0, 1).mul(lp(a, 0, 3).exp())), [0]),
        "both weigh": (lambda b, a: mean(b, lp(a, 0, 1).mul(lp(a, 2, 3)).tanh().mul(lp(a, 2, 3).exp())), [0, 2]),
        "three": (lambda b, a: mean(b, lp(a, 0, 1).mul(lp(a, 2, 3).exp()).mul(lp(a, 0, 3))), [0, 2]),
        "weight and a temperature": (lambda b, a: mean(b, scaled(b, a[0], 0.5).token_log_prob(a[1], "vocab").mul(scaled(b, a[2], 2.0).token_log_prob(a[3], "vocab").exp())), [0, 2]),
    }[name]


ENTANGLED = ["weight", "product of losses", "product of sequences", "preference", "two token sets", "both weigh", "three", "weight and a temperature"]


def entangled_program(name, dtype, s=2, n=3, vocab=40):
    body, wrt = entangled(name)
    logits, tok = T.spec(dtype, s=s, n=n, vocab=vocab), T.spec("i32", s=s, n=n)
    return T.define("entangled", [logits, tok, logits, tok], body), wrt


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("name", ENTANGLED)
def test_log_probabilities_in_each_others_slopes_plan(cpu_session, name, dtype):
    program, wrt = entangled_program(name, dtype)
    for derived in (program.value_and_grad(wrt), program.grad(wrt), program.value_and_grad(wrt[:1])):
        calls = token_calls(plan_lines(cpu_session, derived))
        # every value and every gradient in one kernel each at the most
        assert 2 <= len(calls) <= 6, calls


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [(2, 3, 40), (7, 45, 5003), (3, 101, 33001)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("name", ENTANGLED)
def test_log_probabilities_in_each_others_slopes(gpu_session, name, dtype, sizes):
    """A log-probability of size L is off by step + L / 2^24; a product or an exponential of two of them by the sum of what they are
    off by, relative to their sizes; what follows are sums of s * n terms.  All of it relative to the largest value of its kind."""
    s, n, vocab = sizes
    rng = np.random.default_rng(vocab)
    program, wrt = entangled_program(name, dtype, s, n, vocab)
    xs = [stored(dtype, 2.0 * rng.standard_normal((s, n, vocab))) for _ in range(2)]
    toks = [rng.integers(-1, vocab + 1, (s, n)).astype(np.int32) for _ in range(2)]
    inputs = [xs[0], toks[0], xs[1], toks[1]]
    derived = program.value_and_grad(wrt)
    got, want = run(gpu_session, derived, inputs), oracle.run(derived.wire, inputs, mode="f64")
    top = 2.0 * max(np.abs(exactly(dtype, x)).max() for x in xs)
    step = 2 * max(p_error(2.0 * exactly(dtype, x)) for x in xs) + 16 * U["f32"] * (top + np.log(vocab) + 1) + (s * n + 64) * U["f32"]
    # tanh(p q) with p q above 9 is 1 to f32: its slope 1 - t * t, exactly 4 e^(-2 p q) or less, comes out of two roundings at the size
    # of one (t within two more) and is off by up to 4 * 2^-24 whatever is left of it.  It multiplies p e^q / 16 or
    # q e^q / 16, with e^q <= 1 and |p|, |q| <= 2 top + log(vocab).
    saturated = 4 * U["f32"] * (2 * top + np.log(vocab)) / 16 if name == "both weigh" else 0.0
    for g, w in zip(got, want):
        w = w.reshape(g.shape)
        # the log-probabilities themselves enter the slopes: errors of size step * L relative to products of size L
        close(g, w, 4 * step * (np.abs(w) + np.abs(w).max()) * (1 + np.log(vocab)) + saturated + (U[dtype] if g.ndim else 0) * np.abs(w))


def random_loss(seed):
    """One to four terms of size one at most on log-probabilities of one or two logits tensors, plain or scaled, under one or two sets of
    tokens: means, saturated ones, products of two, whole sequences, squares of the logits."""
    rng = np.random.default_rng(7000 + seed)
    pick = lambda *xs: xs[rng.integers(len(xs))]  # noqa: E731
    s, n, vocab = pick(1, 2, 5), pick(1, 3, 17, 64), pick(2, 33, 130, 1003, 9001)
    tensors, sets = pick(1, 2), pick(1, 2)
    views = [(i, pick(None, 0.5, 3.0, -1.0, "cap")) for i in rng.integers(0, tensors, 3)]
    terms = [(pick("mean", "tanh", "product", "weight", "sequence", "squares"), views[rng.integers(3)], int(rng.integers(sets)), views[rng.integers(3)], int(rng.integers(sets)))
             for _ in range(rng.integers(1, 5))]

    def body(b, a):
        logits, toks = a[:tensors], a[tensors:]
        number = lambda x: b.scalar("f32", x)  # noqa: E731

        def lp(view, tok):
            x = logits[view[0]]
            y = x if view[1] is None else soft_capped(b, x) if view[1] == "cap" else scaled(b, x, view[1])
            return y.token_log_prob(toks[tok], "vocab")
        total = number(0.0)
        for kind, v1, t1, v2, t2 in terms:
            if kind == "squares":
                x = logits[v1[0]]
                term = x.mul(x).sum(["s", "n", "vocab"]).mul(number(1.0 / (16 * s * n * vocab)))
            elif kind == "sequence":
                term = lp(v1, t1).sum("n").mul(number(1.0 / (32 * n))).tanh().sum("s").mul(number(1.0 / s))
            else:
                x = lp(v1, t1)
                x = {"mean": lambda: x.mul(number(1.0 / 32)), "tanh": lambda: x.mul(number(0.25)).tanh(), "product": lambda: x.mul(lp(v2, t2)).mul(number(1.0 / 1024)),
                     "weight": lambda: x.mul(lp(v2, t2).exp()).mul(number(1.0 / 32))}[kind]()
                term = x.sum(["s", "n"]).mul(number(1.0 / (s * n)))
            total = total.add(term)
        return total
    specs = [T.spec("f32", s=s, n=n, vocab=vocab)] * tensors + [T.spec("i32", s=s, n=n)] * sets
    inputs = [2.0 * rng.standard_normal((s, n, vocab)).astype(np.float32) for _ in range(tensors)] + [rng.integers(-1, vocab + 1, (s, n)).astype(np.int32) for _ in range(sets)]
    return T.define("random", specs, body), inputs, list(range(tensors)), (s, n, vocab)


@pytest.mark.parametrize("seed", range(64))
def test_random_losses_plan(cpu_session, seed):
    program, _, wrt, _ = random_loss(seed)
    for derived in (program.value_and_grad(wrt), program.grad(wrt[:1])):
        cpu_session.release(cpu_session.compile(derived))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(64))
def test_random_losses_match_the_oracle(gpu_session, seed):
    """At most four terms; each is at most one and has a slope of at most 1 / (s n) per log-probability, times a factor of at most 3 on the
    way to the logits, and log-probabilities of size up to 32 enter the slopes divided by at least that."""
    program, inputs, wrt, (s, n, vocab) = random_loss(seed)
    derived = program.value_and_grad(wrt)
    got, want = run(gpu_session, derived, inputs), oracle.run(derived.wire, inputs, mode="f64")
    logits = [3.0 * inputs[i].astype(np.float64) for i in wrt]
    step = 2 * max(p_error(x) for x in logits) + 16 * U["f32"] * (max(np.abs(x).max() for x in logits) + np.log(vocab) + 1) + (s * n + vocab + 64) * U["f32"]
    close(got[0].reshape(()), float(want[0].reshape(-1)[0]), 4 * step * 4)
    for g, w in zip(got[1:], want[1:]):
        w = w.reshape(g.shape)
        close(g, w, 4 * step * 4 * 3 / (s * n) + U["f32"] * np.abs(w))


# ---------------------------------------------------------------------------------------------
# planning takes as long as a program is, not as it would be written out without shared values
# ---------------------------------------------------------------------------------------------
@pytest.mark.timeout(120)
@pytest.mark.parametrize("depth", [14, 40])
def test_deep_shared_expressions_plan_in_time(cpu_session, depth):
    """y -> y * tanh(y) read back without sharing has 2^depth leaves."""
    def updates(b, a):
        y = a[1]
        for _ in range(depth):
            y = y.mul(y)
        return b.scalar("f32", 0.0).broadcast(v=5, d=8).scatter_add(a[0], y, "v")

    def loss(b, a):
        y = a[0].token_log_prob(a[1], "vocab")
        for _ in range(depth):
            y = y.mul(y.tanh())
        return y.sum("n")
    for program in (T.define("updates", [T.spec("i32", n=6), T.spec("f32", n=6, d=8)], updates),
                    T.define("loss", [T.spec("f32", n=6, vocab=40), T.spec("i32", n=6)], loss).value_and_grad([0])):
        cpu_session.release(cpu_session.compile(program))


# ---------------------------------------------------------------------------------------------
# the streaming kernel
# ---------------------------------------------------------------------------------------------
def streaming_source(session):
    specs = [T.spec("bf16", n=4096, vocab=131072), T.spec("i32", n=4096)]
    compiled = session.compile(T.define("ce", specs, lambda b, a: nn.cross_entropy(a[0], a[1], "vocab")).value_and_grad([0]))
    sources = [text for _, text, _ in compiled.kernels() if "cp.async.bulk" in text]
    session.release(compiled)
    assert len(sources) == 1
    return sources[0]


def test_every_warp_of_the_streaming_kernel_reports_a_wait_that_gave_up(cpu_session):
    """Every warp raises the session's status word after its own last wait, the producer's and each consumer's: the others may
    have ended before a wait runs out.  (No test makes one run out on a device: that would take a kernel that hangs.)"""
    source = streaming_source(cpu_session)
    producer, consumers = source[source.index("KERNEL(const XT*"):].split("  // Consumers.")
    for part in (producer, consumers):
        last_wait = max(part.rindex("wait_for(&"), part.rindex("passed(") if "passed(" in part else 0)
        assert "*gave_up) atomicExch(status, 1);" in part[last_wait:]
    assert source.count("atomicExch(status, 1)") == 2


# ---------------------------------------------------------------------------------------------
# rows where the model is sure of its token
# ---------------------------------------------------------------------------------------------
def sure_rows(dtype, n, vocab, gap, seed):
    """Logits of deviation 2.5 with one token `gap` above their mean, at the ends of the row and in between"""
    rng = np.random.default_rng(seed)
    x = 2.5 * rng.standard_normal((n, vocab))
    tok = rng.integers(0, vocab, (n,)).astype(np.int32)
    tok[:4] = [0, 1, vocab // 2, vocab - 1]
    x[np.arange(n), tok] = gap
    return stored(dtype, x), tok


def sure_error(gap, p):
    """What log p of such a token may be off by.  Its own term: the token lies at most 5.5 above its reference, an exponent below 8 is
    rounded by at most half a step of [4, 8) (2^-22, in units of log2), log2(e) is off by 1.4e-8 relative, ex2 by 2^-22.  The
    sum: fifteen additions at the size of the total, and terms up to 45 below it, off by 45 * log2(e) * 2^-24 + 2^-22 each,
    which are 1 - p of it.  The logarithm, at most 5.5: half a step of [4, 8) is 2^-22, and the rounding of the difference.
    40 above: the reference is the token itself, and the other terms add up to less than half a step of one, so nothing is added
    to a term of exactly one: ex2 near zero and two roundings."""
    if gap >= 40:
        return 2.0 ** -22 + 2 * U["f32"]
    own = 2.0 ** -22 * np.log(2) + 5.5 * 1.4e-8 + 2.0 ** -22
    return own + 15 * U["f32"] + (1 - p) * (45 * 1.4427 * U["f32"] + 2.0 ** -22) + 2.0 ** -22 + U["f32"]


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [18.0, 25.0, 32.0, 40.0])
@pytest.mark.parametrize("dtype,n,vocab", [("bf16", 40, 131072), ("f32", 40, 300007), ("f16", 700, 50001), ("bf16", 300, 131072), ("f32", 310, 32003), ("bf16", 60, 5003)])
def test_log_probabilities_near_zero(gpu_session, dtype, n, vocab, gap):
    """Few rows are held in registers, split over a cluster or read in chunks; more than two per SM pass through shared memory where a
    gradient is asked for; a slope over all rows takes the kept sums."""
    x, tok = sure_rows(dtype, n, vocab, gap, int(gap) + n)
    want, p, hot, _ = log_prob_of(exactly(dtype, x), tok)
    at = np.arange(n), tok
    p_tok = p[at]
    allowed = sure_error(gap, p_tok)
    specs = [T.spec(dtype, n=n, vocab=vocab), T.spec("i32", n=n)]

    def value(b, a):
        return a[0].token_log_prob(a[1], "vocab")

    def total(b, a):
        return value(b, a).sum("n")

    def sequence(b, a):
        return value(b, a).sum("n").mul(b.scalar("f32", 2.0 ** -20)).tanh()
    got = run(gpu_session, T.define("value", specs, value), [x, tok])[0]
    assert np.all(got <= 0)
    close(got, want, allowed)
    # at the token the gradient is 1 - p, which is what log p has lost
    for body, slope in ((total, 1.0), (sequence, 2.0 ** -20)):
        grad = run(gpu_session, T.define("loss", specs, body).grad([0]), [x, tok])[0]
        exact = slope * (1 - p_tok)
        # the slope of the whole sequence is 2^-20 * (1 - tanh(2^-20 * sum)^2): within 2^-24 of 2^-20 for a sum below 2^8
        assert np.abs(want).sum() < 2.0 ** 8
        close(grad[at], exact, slope * allowed + (U[dtype] + 2.0 ** -20 + 4 * U["f32"]) * exact + TINY[dtype])


# ---------------------------------------------------------------------------------------------
# the largest vocabularies
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 300])
def test_elements_of_the_longest_rows_are_counted_in_32_bits(cpu_session, dtype, n):
    def kernels(vocab, body):
        specs = [T.spec(dtype, n=n, vocab=vocab), T.spec("i32", n=n)]
        compiled = cpu_session.compile(T.define("long", specs, body).grad([0]))
        sources = [text for _, text, _ in compiled.kernels() if "#define VOCAB" in text]
        cpu_session.release(compiled)
        return sources
    bodies = [lambda b, a: a[0].token_log_prob(a[1], "vocab").sum("n"), lambda b, a: a[0].token_log_prob(a[1], "vocab").sum("n").tanh()]
    for body in bodies:
        for source in kernels(2 ** 31 - 2 ** 22, body):
            number = lambda name: int(source.split("#define %s " % name)[1].split("\n")[0])  # noqa: E731,B023
            e, vocab = number("E"), number("VOCAB")
            vectors = vocab // e             # rows of whole vectors
            if "#define CHUNK " in source:   # whole chunks of one row
                reach = -(-vectors // number("CHUNK")) * number("CHUNK")
            else:                            # whole chunks of every part
                reach = number("PARTS") * number("CHUNKS") * number("TPR") * number("VPT")
            assert vectors <= reach and (reach + 1) * e < 2 ** 31
        for vocab in (2 ** 31 - 2 ** 21, 2 ** 31 - 2 ** 20):
            with pytest.raises(T.SessionError) as err:
                kernels(vocab, body)
            assert err.value.name == "compile_failed" and "not supported" in err.value.message
