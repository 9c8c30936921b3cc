"""Categorical distribution given by logits: one row of k unnormalised log-weights per observation (the reference's
categorical.py takes one probability vector for all observations; there is no logits form in it).

Logits have shape (..., k) in float64, float32, float16 or bfloat16, any strides; arithmetic and values (log-density, total)
are float64 for float64 logits and float32 otherwise.  Inputs are torch CUDA tensors (torch results, nothing synchronises)
or NumPy arrays (NumPy results).  Gradients are calls of their own here: nothing is recorded for autograd, which sees a write to
`out` and no more.  csrc/m355_logits.hip."""

from ._logits import adjust as _adjust
from ._logits import adjust_grad as _adjust_grad
from ._logits import logpdf as _logpdf
from ._logits import sum_logpdf as _sum_logpdf


def logpdf(x, logits):
    """Log-density of the observations x, which broadcast to logits.shape[:-1]: logits[x] - log sum exp(logits).  -inf where
    x is no integer in [0, k) and where every logit of the row is -inf; NaN where the row holds NaN or +inf."""
    return _logpdf(x, logits)


def sum_logpdf(x, logits, weights=None):
    """sum(weights * logpdf(x, logits)), added in float64 in a fixed order.  weights broadcast to logits.shape[:-1] (None: 1);
    a row of weight 0 (padding) counts as 0 whatever it and its observation hold."""
    return _sum_logpdf(x, logits, weights, False)[0]


def sum_logpdf_grad(x, logits, weights=None, out=None):
    """(sum_logpdf(x, logits, weights), [None, its gradient with respect to the logits]); the gradient,
    weights * ([v == x] - softmax(logits)[v]), has the logits' shape and dtype and is 0 in rows of weight 0, rows whose x is
    no category and rows that are all -inf.  out: where the gradient goes; it may be the logits themselves."""
    total, g = _sum_logpdf(x, logits, weights, True, out)
    return total, [None, g]


def adjust(logits, history=None, lengths=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias=None,
           temperature=1.0, mask=None, out=None):
    """Logits as they are scored (by logpdf) or drawn from: with c_all and c_gen the number of times category v stands in
    history[..., :lengths] and history[..., prompt_lengths:lengths],

        s = logits;  where c_all > 0:  s = s / repetition if s > 0 else s * repetition
        s = s - frequency * c_gen - presence * (c_gen > 0);  s = s + bias;  s = s / temperature;  s = -inf where not allowed

    history: integer ids (..., n), those outside [0, k) are skipped (padding); lengths, prompt_lengths: integers per row
    (default n and 0; clamped to [0, n]).  repetition, presence, frequency, temperature: numbers or arrays per row.  bias:
    (k,) or (..., k), of the logits' dtype or float32 (other types are converted).  mask: truth values (k,) or (..., k), or
    int32 words (..., ceil(k / 32)) in which category v is bit v % 32 of word v // 32; true / 1 = allowed.  A row that allows
    nothing is all -inf.  out: where the result goes; it may be the logits themselves.  Arrays with leading axes broadcast to
    logits.shape[:-1]."""
    return _adjust(logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias, temperature, mask, out)


def adjust_grad(g, logits, history=None, lengths=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0,
                bias=None, temperature=1.0, mask=None):
    """(gradient with respect to the logits, with respect to the bias or None) of adjust(logits, ...) for the gradient g of
    its result (g is converted to the logits' dtype); each has the shape and dtype of its argument.  Penalties, temperature
    and mask are data.  A bias that rows share, all of them or along some of their axes, gets the sum over them, added in
    float64 in a fixed order.  Not allowed: 0, whatever g holds there."""
    return _adjust_grad(g, logits, history, lengths, prompt_lengths, repetition, presence, frequency, bias, temperature, mask)
