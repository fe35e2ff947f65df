"""The token side of a language model, recorded with the operations of `accy_b200.tensor`: embedding
lookup and its gradient, and losses on the log-probabilities of given tokens.

Each function takes and returns recorded `tensor.Value`s, so it is used inside the body of a
`tensor.define`; gradients come from `value_and_grad` like those of any other program, and a loss and
its gradient with respect to the logits are one pass over the logits.

Batches are padded two ways, which may be mixed: a token outside [0, extent) (-1, say) looks up zeros,
adds nothing to a gradient and counts in no loss, and a zero in `mask` (f32 with some or all of the
tokens' axes, 1 where a token counts) keeps a position out of a loss.  What the other inputs hold at
such a position has no influence, be it NaN or infinite, and its row of the logits' gradient is zero.
A loss over no position at all is 0.
"""
from .tensor import TensorError


def embedding(table, tokens, axis, scale=None):
    """Rows of `table` along `axis`, one for each of `tokens`, times the number `scale`."""
    rows = table.gather(tokens, axis)
    return rows if scale is None else rows.mul(rows.builder.scalar(rows.ty.dtype, scale))


def embedding_grad(tokens, grad, axis, extent, scale=None):
    """The gradient of `embedding` with respect to its table, from `grad`, the gradient of its result:
    [axis = extent, the axes of `grad` that `tokens` lacks], typed like `grad`."""
    b, dtype = grad.builder, grad.ty.dtype
    known = [name for name, _ in tokens.ty.dims]
    rest = [d for d in grad.ty.dims if d[0] not in known]
    zeros = b.scalar(dtype, 0.0).broadcast(**dict([(axis, extent)] + rest))
    return zeros.scatter_add(tokens, grad if scale is None else grad.mul(b.scalar(dtype, scale)), axis)


_LARGEST = {"i8": 127, "i16": 32767, "i32": 2**31 - 1, "i64": 2**63 - 1, "u8": 255, "u16": 65535, "u32": 2**32 - 1,
            "u64": 2**64 - 1}


def _counted(logits, tokens, axis, mask):
    """(f32 weight of every position, whether it counts): the mask where the token is in the vocabulary, 0 elsewhere."""
    b, dtype = logits.builder, tokens.ty.dtype
    extent = dict(logits.ty.dims).get(axis)
    if extent is None:
        raise TensorError("AxisNotFound")
    if dtype not in _LARGEST:
        raise TensorError("NonIntegerDType")
    zero = b.scalar("f32", 0.0)
    weight = b.scalar("f32", 1.0) if mask is None else mask
    if extent <= _LARGEST[dtype]:   # otherwise no number of the type is past the end
        weight = tokens.compare("lt", b.scalar(dtype, extent)).select(weight, zero)
    weight = tokens.compare("ge", b.scalar(dtype, 0)).select(weight, zero)
    return weight, weight.compare("ne", zero)


def _mean(values, weight):
    """sum(weight * values) / max(sum(weight), 1)"""
    axes = [name for name, _ in values.ty.dims]
    return values.mul(weight).sum(axes).div(weight.sum(axes).max(values.builder.scalar("f32", 1.0)))


def cross_entropy(logits, tokens, axis, mask=None):
    """The mean of -log p(token) over the positions that count, an f32 number; p is the softmax of
    `logits` (f32, bf16 or f16) along `axis`, which `tokens` lacks."""
    weight, counts = _counted(logits, tokens, axis, mask)
    zero = logits.builder.scalar("f32", 0.0)
    return _mean(counts.select(logits.token_log_prob(tokens, axis), zero).neg(), weight)


def policy_loss(logits, tokens, axis, old, reference, advantage, mask=None, clip=0.2, kl=0.0):
    """The clipped policy loss with a KL term, an f32 number: the mean, over the positions that count, of

        kl * (exp(d) - d - 1) - min(r * a, min(max(r, 1 - clip), 1 + clip) * a)

    with r = exp(log p - old) against the log-probabilities the tokens were drawn with, d = reference -
    log p against those of a fixed model, and the advantage a.  `old` and `reference` are f32 with the
    tokens' axes, `advantage` f32 with some or all of them.  Where r * a and the clipped product are
    equal the gradient is that of r * a."""
    b = logits.builder
    zero, one = b.scalar("f32", 0.0), b.scalar("f32", 1.0)
    weight, counts = _counted(logits, tokens, axis, mask)
    log_prob, old, reference, advantage = (counts.select(x, zero) for x in (logits.token_log_prob(tokens, axis), old, reference, advantage))
    ratio = log_prob.sub(old).exp()
    held = ratio.max(b.scalar("f32", 1.0 - clip)).min(b.scalar("f32", 1.0 + clip))
    loss = ratio.mul(advantage).min(held.mul(advantage)).neg()
    if kl:
        gap = reference.sub(log_prob)
        loss = loss.add(gap.exp().sub(gap).sub(one).mul(b.scalar("f32", kl)))
    return _mean(loss, weight)
