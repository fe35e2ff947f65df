"""The token side of a language model's step: looking token embeddings up, the gradient of that
lookup, the log-probability of given tokens, and two losses built on it with their gradients.

`run` computes each in its plain form (elementary torch operations in 32 bits, rounded once at the
end), or, where `own` is true, as one launch of a program recorded and compiled with `accy_b200`.

    embedding       out[t, :]  = scale * table[token[t], :]
    embedding_grad  out[v, :]  = scale * sum over the t with token[t] = v of grad[t, :]
    token_log_prob  out[t]     = logits[t, token[t]] - log(sum_v exp(logits[t, v]))
    cross_entropy   loss       = -sum_t mask[t] * log_prob[t] / max(sum_t mask[t], 1), and d loss / d logits
    policy_loss     loss       = sum_t mask[t] * (kl * (exp(d) - d - 1) - min(r * a, clip(r) * a)) / max(sum_t mask[t], 1)
                                 with r = exp(log_prob - old), clip(r) = min(max(r, 1 - c), 1 + c), d = reference - log_prob,
                                 a the advantage of t's sequence; and d loss / d logits

A token outside the vocabulary (-1 pads the batches) reads zeros, adds nothing to a gradient and has
the log-probability zero.  Where the mask is zero nothing enters a loss and the gradient's row is zero.
"""
import math

import torch

own = False

DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
INDEX = {"i32": torch.int32, "i64": torch.int64}
CLIP, KL = 0.2, 0.05


# ---- the cases -----------------------------------------------------------------------------
def listed():
    return [
        # one new token for each of 16 sequences of a serving batch: the smallest call
        {"name": "embedding_step", "op": "embedding", "dtype": "bf16", "index": "i32", "batch": 16, "seq": 1, "vocab": 131072, "dim": 4096},
        # the tokens of a training step
        {"name": "embedding_train", "op": "embedding", "dtype": "bf16", "index": "i32", "batch": 8, "seq": 4096, "vocab": 32768, "dim": 4096},
        # odd sizes in 32 bits, with the 64-bit token numbers that tokenizers hand out
        {"name": "embedding_odd", "op": "embedding", "dtype": "f32", "index": "i64", "batch": 7, "seq": 1365, "vocab": 50001, "dim": 1001},
        # the gradient of a fine-tuning step: few tokens, most rows of the table untouched
        {"name": "embedding_grad_tune", "op": "embedding_grad", "dtype": "bf16", "index": "i32", "batch": 4, "seq": 512, "vocab": 32768, "dim": 2048},
        # odd sizes in 32 bits; a few tokens make up most of the batch
        {"name": "embedding_grad_odd", "op": "embedding_grad", "dtype": "f32", "index": "i64", "batch": 9, "seq": 1111, "vocab": 10007, "dim": 513},
        # the gradient of a large training step
        {"name": "embedding_grad_train", "op": "embedding_grad", "dtype": "bf16", "index": "i32", "batch": 16, "seq": 4096, "vocab": 131072, "dim": 4096},
        # the log-probability of one sampled token for each of 8 sequences
        {"name": "log_prob_step", "op": "token_log_prob", "dtype": "bf16", "index": "i32", "batch": 8, "seq": 1, "vocab": 131072, "dim": 0},
        # scoring whole sequences against a vocabulary of odd size
        {"name": "log_prob_score", "op": "token_log_prob", "dtype": "f16", "index": "i32", "batch": 4, "seq": 1023, "vocab": 50001, "dim": 0},
        # a small training step in 32 bits
        {"name": "cross_entropy_f32", "op": "cross_entropy", "dtype": "f32", "index": "i64", "batch": 3, "seq": 341, "vocab": 32003, "dim": 0},
        # a large training step: the largest call
        {"name": "cross_entropy_train", "op": "cross_entropy", "dtype": "bf16", "index": "i32", "batch": 8, "seq": 1024, "vocab": 131072, "dim": 0},
        # policy training on a few short answers
        {"name": "policy_short", "op": "policy_loss", "dtype": "bf16", "index": "i32", "batch": 4, "seq": 64, "vocab": 32768, "dim": 0},
        # policy training on a group of long answers
        {"name": "policy_group", "op": "policy_loss", "dtype": "bf16", "index": "i32", "batch": 8, "seq": 777, "vocab": 65536, "dim": 0},
    ]


def draw(rng):
    def spread(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(lo, min(hi, n | 1 if rng.random() < 0.4 else n))

    op = rng.choice(["embedding", "embedding_grad", "token_log_prob", "cross_entropy", "policy_loss"])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"] if op in ("embedding", "token_log_prob") else ["bf16", "bf16", "f32"])
    case = {"op": op, "dtype": dtype, "index": rng.choice(["i32", "i64"]), "batch": spread(1, 32), "seq": 1, "vocab": spread(1000, 200000), "dim": 0}
    case["seq"] = spread(1, 4096)
    if op.startswith("embedding"):
        case["dim"] = spread(64, 8192)
        while case["vocab"] * case["dim"] > 1 << 29 or case["batch"] * case["seq"] * case["dim"] > 1 << 28:
            key = max(("vocab", "dim", "seq", "batch"), key=lambda k: case[k])
            case[key] = max(1, case[key] // 2)
    else:
        most = 1 << 30 if dtype != "f32" else 1 << 29
        while case["batch"] * case["seq"] * case["vocab"] > most:
            key = "seq" if case["seq"] >= case["batch"] else "batch"
            case[key] = max(1, case[key] // 2)
    return case


def work(case):
    tokens, vocab, dim, size = case["batch"] * case["seq"], case["vocab"], case["dim"], SIZE[case["dtype"]]
    ids = tokens * (4 if case["index"] == "i32" else 8)
    if case["op"] == "embedding":
        return {"bytes": ids + min(tokens, vocab) * dim * size + tokens * dim * size, "flops": tokens * dim}
    if case["op"] == "embedding_grad":
        return {"bytes": ids + tokens * dim * size + vocab * dim * size, "flops": 2 * tokens * dim}
    if case["op"] == "token_log_prob":
        return {"bytes": ids + tokens * vocab * size + 4 * tokens, "flops": 4 * tokens * vocab}
    rows = 4 * tokens if case["op"] == "cross_entropy" else 12 * tokens + 4 * case["batch"]
    return {"bytes": ids + rows + 2 * tokens * vocab * size + 4, "flops": 8 * tokens * vocab}


# ---- inputs --------------------------------------------------------------------------------
def scale_of(case):
    """A whole number near the square root of the width, which every element type holds exactly."""
    return float(max(1, round(math.sqrt(case["dim"]))))


def log_probs(logits, token):
    """The tokens' log-probabilities in 64 bits, some rows at a time."""
    flat, ids = logits.reshape(-1, logits.shape[-1]), token.reshape(-1).long()
    out = torch.empty(flat.shape[0], dtype=torch.float64, device=flat.device)
    step = max(1, (1 << 26) // flat.shape[1])
    for i in range(0, flat.shape[0], step):
        x = flat[i:i + step].double()
        at = ids[i:i + step].clamp(0, flat.shape[1] - 1).unsqueeze(1)
        out[i:i + step] = x.gather(1, at).squeeze(1) - torch.logsumexp(x, 1)
    return torch.where((ids >= 0) & (ids < flat.shape[1]), out, torch.zeros_like(out)).reshape(token.shape)


def inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    batch, seq, vocab, dim, dtype = case["batch"], case["seq"], case["vocab"], case["dim"], DTYPE[case["dtype"]]

    def normal(*shape, to=torch.float32):
        return torch.empty(shape, dtype=to, device="cuda").normal_(generator=g)

    # few tokens are frequent and most are rare
    token = (vocab * torch.rand(batch, seq, generator=g, device="cuda", dtype=torch.float64) ** 4).to(INDEX[case["index"]])
    # sequences of different lengths, padded at the end; single tokens are all there
    length = torch.randint(seq // 2, seq + 1, (batch, 1), generator=g, device="cuda")
    if seq > 1 and batch > 2:
        length[1] = 0
    if seq == 1:
        length = torch.ones_like(length)
    there = torch.arange(seq, device="cuda") < length
    token = torch.where(there, token, torch.full_like(token, -1))
    if case["op"] == "embedding":
        return {"table": normal(vocab, dim, to=dtype), "token": token}
    if case["op"] == "embedding_grad":
        return {"token": token, "grad": normal(batch, seq, dim, to=dtype)}
    logits = normal(batch, seq, vocab, to=dtype).mul_(2.5)
    # the model has learned something: the tokens that are there are likelier than others
    at = token.long().clamp(0, vocab - 1).unsqueeze(2)
    logits.scatter_add_(2, at, torch.full(at.shape, 4.0, dtype=dtype, device="cuda"))
    if case["op"] == "token_log_prob":
        return {"logits": logits, "token": token}
    mask = there.float()
    if case["op"] == "cross_entropy":
        return {"logits": logits, "token": token, "mask": mask}
    now = log_probs(logits, token)
    off = 0.15 * normal(batch, seq).double()
    # no ratio next to a border of the clipping, where one rounding decides about a whole row
    ratio = torch.exp(off)
    off = torch.where(((ratio - (1 - CLIP)).abs() < 0.01) | ((ratio - (1 + CLIP)).abs() < 0.01), torch.zeros_like(off), off)
    return {"logits": logits, "token": token, "old": (now - off).float(), "reference": (now + 0.3 * normal(batch, seq).double()).float(),
            "advantage": normal(batch), "mask": mask}


def prepare(case, seed):
    state = {"case": case, "inputs": inputs(case, seed)}
    if own:
        state["plan"] = plan(case)
    return state


# ---- the framework's operators -----------------------------------------------------------------
def plan(case):
    """The program of the case, recorded and compiled, with the buffers its outputs go to."""
    from accy_b200 import nn, tensor

    dtype, index = case["dtype"], case["index"]
    batch, seq, vocab, dim = case["batch"], case["seq"], case["vocab"], case["dim"]
    token = tensor.spec(index, batch=batch, seq=seq)
    row = tensor.spec("f32", batch=batch, seq=seq)
    logits = tensor.spec(dtype, batch=batch, seq=seq, vocab=vocab)
    if case["op"] == "embedding":
        program = tensor.define("embedding", [tensor.spec(dtype, vocab=vocab, dim=dim), token],
                                lambda b, a: nn.embedding(a[0], a[1], "vocab", scale=scale_of(case)))
        shapes = [((batch, seq, dim), DTYPE[dtype])]
    elif case["op"] == "embedding_grad":
        program = tensor.define("embedding_grad", [token, tensor.spec(dtype, batch=batch, seq=seq, dim=dim)],
                                lambda b, a: nn.embedding_grad(a[0], a[1], "vocab", vocab, scale=scale_of(case)))
        shapes = [((vocab, dim), DTYPE[dtype])]
    elif case["op"] == "token_log_prob":
        program = tensor.define("token_log_prob", [logits, token], lambda b, a: a[0].token_log_prob(a[1], "vocab"))
        shapes = [((batch, seq), torch.float32)]
    elif case["op"] == "cross_entropy":
        program = tensor.define("cross_entropy", [logits, token, row],
                                lambda b, a: nn.cross_entropy(a[0], a[1], "vocab", mask=a[2])).value_and_grad([0])
        shapes = [((), torch.float32), ((batch, seq, vocab), DTYPE[dtype])]
    else:
        program = tensor.define("policy_loss", [logits, token, row, row, tensor.spec("f32", batch=batch), row],
                                lambda b, a: nn.policy_loss(a[0], a[1], "vocab", old=a[2], reference=a[3], advantage=a[4], mask=a[5],
                                                            clip=CLIP, kl=KL)).value_and_grad([0])
        shapes = [((), torch.float32), ((batch, seq, vocab), DTYPE[dtype])]
    return {"cuda": tensor.Cuda(program, device=torch.cuda.current_device()),
            "outputs": [torch.empty(shape, dtype=dtype, device="cuda") for shape, dtype in shapes]}


def launch(plan, given):
    # 1 names the legacy default stream, which torch writes as 0
    stream = torch.cuda.current_stream().cuda_stream or 1
    plan["cuda"].launch_device([x.data_ptr() for x in given], [x.data_ptr() for x in plan["outputs"]], stream)
    return plan["outputs"]


# ---- the plain forms -----------------------------------------------------------------------
def plain_embedding(case, table, token):
    there = (token >= 0) & (token < case["vocab"])
    rows = table[token.long().clamp(0, case["vocab"] - 1)].float() * scale_of(case)
    return [torch.where(there.unsqueeze(-1), rows, torch.zeros_like(rows)).to(table.dtype)]


def plain_embedding_grad(case, token, grad):
    ids = token.reshape(-1).long()
    there = (ids >= 0) & (ids < case["vocab"])
    rows = torch.where(there.unsqueeze(1), grad.reshape(-1, case["dim"]).float(), 0.0)
    out = torch.zeros(case["vocab"], case["dim"], dtype=torch.float32, device="cuda")
    out.index_add_(0, ids.clamp(0, case["vocab"] - 1), rows)
    return [(out * scale_of(case)).to(grad.dtype)]


def plain_log_prob(logits, token):
    """The log-probabilities, the probabilities, the token's place in the row, and whether it is in the vocabulary."""
    x = logits.float()
    there = (token >= 0) & (token < x.shape[-1])
    at = token.long().clamp(0, x.shape[-1] - 1).unsqueeze(-1)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    log_prob = (x.gather(-1, at) - top - torch.log(total)).squeeze(-1)
    return torch.where(there, log_prob, torch.zeros_like(log_prob)), e / total, at, there


def plain_grad(logits, slope, p, at, there):
    """d loss / d logits, given d loss / d log_prob."""
    slope = torch.where(there, slope, torch.zeros_like(slope)).unsqueeze(-1)
    grad = p * -slope
    return grad.scatter_add_(-1, at, slope).to(logits.dtype)


def plain_cross_entropy(logits, token, mask):
    log_prob, p, at, there = plain_log_prob(logits, token)
    count = mask.sum().clamp(min=1.0)
    loss = -(mask * log_prob).sum() / count
    return [loss, plain_grad(logits, -mask / count, p, at, there)]


def plain_policy_loss(logits, token, old, reference, advantage, mask):
    log_prob, p, at, there = plain_log_prob(logits, token)
    count = mask.sum().clamp(min=1.0)
    a = advantage.unsqueeze(1)
    ratio = torch.exp(log_prob - old)
    free, held = ratio * a, ratio.clamp(1 - CLIP, 1 + CLIP) * a
    d = reference - log_prob
    loss = (mask * (KL * (torch.exp(d) - d - 1) - torch.minimum(free, held))).sum() / count
    slope = mask * (KL * (1 - torch.exp(d)) - torch.where(free <= held, free, torch.zeros_like(free))) / count
    return [loss, plain_grad(logits, slope, p, at, there)]


def run(state):
    case, given = state["case"], state["inputs"]
    if own:
        return launch(state["plan"], list(given.values()))
    if case["op"] == "embedding":
        return plain_embedding(case, given["table"], given["token"])
    if case["op"] == "embedding_grad":
        return plain_embedding_grad(case, given["token"], given["grad"])
    if case["op"] == "token_log_prob":
        return [plain_log_prob(given["logits"], given["token"])[0]]
    if case["op"] == "cross_entropy":
        return plain_cross_entropy(given["logits"], given["token"], given["mask"])
    return plain_policy_loss(**given)


# ---- the definition in 64 bits -----------------------------------------------------------------
def exact(case, seed):
    given, vocab = inputs(case, seed), case["vocab"]
    ids = given["token"].reshape(-1).long()
    known = ((ids >= 0) & (ids < vocab)).double()
    ids = ids * known.long()
    if case["op"] == "embedding":
        rows = given["table"].double()[ids] * known.unsqueeze(1) * scale_of(case)
        return [rows.reshape(case["batch"], case["seq"], case["dim"])]
    if case["op"] == "embedding_grad":
        out = torch.zeros(vocab, case["dim"], dtype=torch.float64, device="cuda")
        out.index_add_(0, ids, given["grad"].double().reshape(-1, case["dim"]) * (known * scale_of(case)).unsqueeze(1))
        return [out]
    log_prob = log_probs(given["logits"], given["token"])
    if case["op"] == "token_log_prob":
        return [log_prob]
    mask = given["mask"].double()
    weight = mask / max(float(mask.sum()), 1.0)
    if case["op"] == "cross_entropy":
        loss, slope = -(weight * log_prob).sum(), -weight
    else:
        a = given["advantage"].double()[:, None]
        ratio = (log_prob - given["old"].double()).exp()
        gap = given["reference"].double() - log_prob
        # past the border on the side where the objective would still grow, the slope is zero
        held = ((a > 0) & (ratio > 1 + CLIP)) | ((a < 0) & (ratio < 1 - CLIP))
        gain = torch.where(held, a * torch.where(a > 0, 1 + CLIP, 1 - CLIP), a * ratio)
        loss = (weight * (KL * (torch.expm1(gap) - gap) - gain)).sum()
        slope = weight * (-KL * torch.expm1(gap) - torch.where(held, torch.zeros_like(gain), a * ratio))
    slope = slope.reshape(-1) * known
    flat = given["logits"].reshape(-1, vocab)
    grad = torch.empty(flat.shape, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 26) // vocab)
    for i in range(0, flat.shape[0], step):
        s = slope[i:i + step, None]
        grad[i:i + step] = torch.softmax(flat[i:i + step].double(), 1) * -s
        grad[i:i + step].scatter_add_(1, ids[i:i + step, None], s)
    return [loss, grad.reshape(given["logits"].shape)]
