"""Plain PyTorch fp32 statements of every op in :mod:`distributed_tensorflow_amd.ops`.

These are (a) the CPU execution path (the framework runs end to end without a
GPU, e.g. the "1 ps + 2 workers on CPU" configuration) and (b) the oracle the
HIP kernels are tested against.  The math transcribes
/root/reference/distributed.py:78-89 and the gradients TensorFlow's autodiff
derives from it (``opt.minimize``, distributed.py:102).
"""
from __future__ import annotations

import functools
import math

import torch

LOSS_REFERENCE = 0   # softmax_cross_entropy_with_logits applied to an already-softmaxed y (distributed.py:81, :86)
LOSS_STANDARD = 1    # cross entropy on the logits


def linear_fwd(x, w, b=None, relu=False, rows=None):
    if rows is not None:
        x = x.index_select(0, rows.long())
    y = x @ w
    if b is not None:
        y = y + b
    return torch.relu(y) if relu else y


def linear_bwd_data(dy, w, act=None):
    """dX = dY @ W^T, masked where the forward activation was not positive (ReluGrad)."""
    dx = dy @ w.t()
    if act is not None:
        dx = torch.where(act > 0, dx, torch.zeros_like(dx))
    return dx


def wgrad(x, dy, rows=None):
    if rows is not None:
        x = x.index_select(0, rows.long())
    return x.t() @ dy, dy.sum(0)


def head(hact, w2, b2, labels, m_train, loss_mode=LOSS_REFERENCE, rows=None, want_dz1=True):
    """Last layer + loss + accuracy + gradients for the first ``m_train`` rows.

    Returns a dict with ``loss_sum`` (sum over training rows, not yet divided by
    the batch size), ``correct`` (training rows), ``post_correct`` (rows
    ``>= m_train``), ``probs``, ``dz2`` [m_train, C] and ``dz1`` [m_train, Hd].
    """
    m_total = hact.shape[0]
    if rows is not None:
        labels = labels.index_select(0, rows[:m_total].long())
    else:
        labels = labels[:m_total]
    z = hact @ w2 + b2
    y = torch.softmax(z, dim=1)
    hit = (y.argmax(1) == labels.argmax(1))
    out = {"probs": y,
           "correct": int(hit[:m_train].sum().item()),
           "post_correct": int(hit[m_train:].sum().item())}
    if m_train == 0:
        out["loss_sum"] = 0.0
        return out
    yt, lt, zt = y[:m_train], labels[:m_train], z[:m_train]
    inv_b = 1.0 / m_train
    if loss_mode == LOSS_REFERENCE:
        logp = torch.log_softmax(yt, dim=1)
        p = torch.softmax(yt, dim=1)
        dy = (p - lt) * inv_b
        dz2 = (dy - (dy * yt).sum(1, keepdim=True)) * yt
    else:
        logp = torch.log_softmax(zt, dim=1)
        dz2 = (yt - lt) * inv_b
    out["loss_sum"] = float(-(lt * logp).sum().item())
    out["loss_rows"] = -(lt * logp).sum(1)
    out["dz2"] = dz2
    if want_dz1:
        out["dz1"] = linear_bwd_data(dz2, w2, hact[:m_train])
    return out


def sgd_apply(param, grad, lr, grad_scale=1.0):
    param.sub_(grad * (lr * grad_scale))
    return param


def adam_apply(param, grad, m, v, lr, beta1, beta2, eps, grad_scale, step):
    """Textbook Adam (identical to torch.optim.Adam without weight decay); ``step`` counts from 1."""
    g = grad * grad_scale
    m.mul_(beta1).add_(g, alpha=1 - beta1)
    v.mul_(beta2).addcmul_(g, g, value=1 - beta2)
    bc1 = 1 - beta1 ** step
    bc2 = 1 - beta2 ** step
    denom = (v.sqrt() / math.sqrt(bc2)).add_(eps)
    param.addcdiv_(m, denom, value=-lr / bc1)
    return param


def truncated_normal(shape, stddev, generator=None, device="cpu"):
    """N(0, stddev) re-sampled until |v| <= 2 stddev (tf.truncated_normal, distributed.py:67-72)."""
    out = torch.empty(shape, dtype=torch.float32, device=device)
    flat = out.view(-1)
    todo = torch.arange(flat.numel(), device=device)
    while todo.numel() > 0:
        cand = torch.randn(todo.numel(), generator=generator, device=device)
        ok = cand.abs() <= 2.0
        flat[todo[ok]] = cand[ok]
        todo = todo[~ok]
    return out * stddev


def softmax_xent(logits, labels, loss_mode=LOSS_STANDARD, grad_scale=None):
    """Loss rows, gradient wrt the logits and hit count of softmax cross-entropy over ``[B, C]`` logits; ``labels`` are
    one-hot / soft rows ``[B, C]`` or class indices ``[B]``.  Same two loss modes as :func:`head`."""
    b, c = logits.shape
    z = logits.float()
    if labels.dim() == 1:
        lab = torch.zeros_like(z)
        ok = (labels >= 0) & (labels < c)
        lab[ok, labels[ok].long()] = 1.0
        am_l = labels.long()
    else:
        lab = labels.float()
        am_l = lab.argmax(1)
    scale = (1.0 / b) if grad_scale is None else grad_scale
    y = torch.softmax(z, 1)
    if loss_mode == LOSS_REFERENCE:
        logp = torch.log_softmax(y, 1)
        p = torch.softmax(y, 1)
        dy = (p - lab) * scale
        dz = (dy - (dy * y).sum(1, keepdim=True)) * y
    else:
        logp = torch.log_softmax(z, 1)
        dz = (y - lab) * scale
    return {"loss_rows": -(lab * logp).sum(1), "dlogits": dz, "correct": int((z.argmax(1) == am_l).sum().item())}


# ------------------------------------------------------------------------------------------- token-model operators
def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None):
    """``(y, h, mean, rstd)`` of layer normalisation over the last axis of ``h = x [+ residual]`` (``h`` as stored)."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    v = h.float()
    mean = v.mean(-1, keepdim=True)
    centred = v - mean
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + eps)
    y = centred * rstd
    if weight is not None:
        y = y * weight.float()
    if bias is not None:
        y = y + bias.float()
    return y.to(x.dtype), h, mean.reshape(-1), rstd.reshape(-1)


def layer_norm_bwd(dy, h, mean, rstd, weight=None, dh=None):
    """``(dx, dweight, dbias)``; the parameters' gradients in float32."""
    cols = h.shape[-1]
    d = dy.float().reshape(-1, cols)
    xhat = (h.float().reshape(-1, cols) - mean[:, None]) * rstd[:, None]
    g = d if weight is None else d * weight.float()
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    if dh is not None:
        dx = dx + dh.float().reshape(-1, cols)
    return dx.to(h.dtype).reshape(dy.shape), (d * xhat).sum(0), d.sum(0)


def philox_words(blocks, seed, step, device="cpu"):
    """``[blocks, 4]`` words (int64 holding 32 bits) of Philox4x32-10 for the counters ``(i, step)`` under key ``seed``."""
    m32 = 0xFFFFFFFF
    i = torch.arange(blocks, dtype=torch.int64, device=device)
    c = [i & m32, i >> 32, torch.full_like(i, step & m32), torch.full_like(i, (step >> 32) & m32)]
    k0, k1 = seed & m32, (seed >> 32) & m32
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57          # modulo 2^64: the sign bit is a bit like the others
        c = [((p1 >> 32) & m32) ^ c[1] ^ k0, p1 & m32, ((p0 >> 32) & m32) ^ c[3] ^ k1, p0 & m32]
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    return torch.stack(c, 1)


def dropout_mask(shape, rate, seed, step, device="cpu"):
    """True where dropout keeps the element: its 16-bit number is at least ``round(rate * 65536)``."""
    n = math.prod(shape)
    w = philox_words(-(-n // 8), seed, step, device)
    u = torch.stack((w & 0xFFFF, w >> 16), 2).reshape(-1)[:n]
    return (u >= int(round(rate * 65536))).reshape(shape)


def dropout(x, rate, seed, step=0, residual=None):
    thr = int(round(rate * 65536))
    scale = 65536.0 / (65536 - thr) if thr < 65536 else 0.0
    kept = dropout_mask(tuple(x.shape), rate, seed, step, x.device)
    y = torch.where(kept, x.float() * scale, torch.zeros((), dtype=torch.float32, device=x.device))
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype)


def _vocab_labels(labels, vocab, ignore_index):
    valid = labels != ignore_index
    lab = torch.where(valid, labels, torch.zeros_like(labels))
    if bool(((lab < 0) | (lab >= vocab)).any()):
        raise IndexError(f"vocab_xent: a label lies outside [0, {vocab}) and is not ignore_index")
    return valid, lab


def _float32_products(f):
    """``f`` without autocast, which would run its products in a lower type."""
    @functools.wraps(f)
    def run(features, *args, **kw):
        with torch.autocast(features.device.type, enabled=False):
            return f(features, *args, **kw)
    return run


@_float32_products
def vocab_xent(features, weight, labels, bias=None, ignore_index=-100, reduction="mean"):
    """``(loss, rows, [hits, rows with a label])`` of softmax cross entropy on ``features @ weight.T + bias``; ``rows`` [4, N]:
    loss, logarithm of the sum of exponentials, largest logit, sum of exponentials relative to it."""
    z = features.float() @ weight.float().t()
    if bias is not None:
        z = z + bias.float()
    valid, lab = _vocab_labels(labels, weight.shape[0], ignore_index)
    lse = torch.logsumexp(z, 1)
    rows = torch.where(valid, lse - z.gather(1, lab[:, None])[:, 0], torch.zeros_like(lse))
    counts = torch.stack([((z.argmax(1) == lab) & valid).sum(), valid.sum()])
    total = rows.sum()
    if reduction == "mean":
        total = total / counts[1].clamp_min(1)
    top = z.amax(1)
    return total, torch.stack((rows, lse, top, torch.exp(z - top[:, None]).sum(1))), counts


@_float32_products
def vocab_xent_bwd(features, weight, labels, bias, lse, counts, ignore_index=-100, reduction="mean", dloss=None):
    """``(dfeatures, dweight, dbias)``; dbias None without a bias."""
    x, w = features.float(), weight.float()
    z = x @ w.t()
    if bias is not None:
        z = z + bias.float()
    valid, lab = _vocab_labels(labels, weight.shape[0], ignore_index)
    g = torch.ones((), device=x.device) if dloss is None else dloss.float().reshape(-1 if reduction == "none" else ())
    if reduction == "mean":
        g = g / counts[1].clamp_min(1)
    g = torch.where(valid, g.expand(x.shape[0]), torch.zeros((), device=x.device))
    dz = torch.exp(z - lse[:, None])
    dz.scatter_add_(1, lab[:, None], torch.full_like(lse, -1.0)[:, None])
    used = (g != 0)[:, None]                       # a row without a gradient may hold anything, also NaN
    dz = torch.where(used, dz * g[:, None], torch.zeros((), device=x.device))
    x = torch.where(used, x, torch.zeros((), device=x.device))
    db = None if bias is None else dz.sum(0).to(bias.dtype)
    return (dz @ w).to(features.dtype), (dz.t() @ x).to(weight.dtype), db


def embedding(ids, table, scale=1.0):
    return (torch.nn.functional.embedding(ids.long(), table).float() * scale).to(table.dtype)


def embedding_bwd(dy, ids, rows, scale=1.0, padding_idx=None):
    flat, d = ids.reshape(-1).long(), dy.float().reshape(-1, dy.shape[-1])
    if padding_idx is not None:
        keep = flat != padding_idx % rows
        flat, d = flat[keep], d[keep]
    out = torch.zeros((rows, dy.shape[-1]), dtype=torch.float32, device=dy.device)
    return (out.index_add_(0, flat, d) * scale).to(dy.dtype)
