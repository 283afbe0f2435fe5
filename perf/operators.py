"""Cases that measure the framework's token-model operators: layer normalisation, dropout, embedding and the
vocabulary-wide softmax cross entropy, each in its plain form and (``own``) through the framework's entry points.

A plain form is elementary torch operations in 32 bits, rounded once at the end.  ``exact`` states the same outputs in
64 bits.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
IGNORE = -100
EPS = 1e-5


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a decoder behind a residual addition: nothing but latency
        dict(name="ln_one_token", op="layer_norm", rows=1, cols=4096, dtype="bf16", residual=True, train=False),
        # a training batch's activations between two blocks
        dict(name="ln_train_batch", op="layer_norm", rows=8192, cols=4096, dtype="bf16", residual=True, train=True),
        # an odd feature width in full precision, ragged row count
        dict(name="ln_train_odd_f32", op="layer_norm", rows=5001, cols=1001, dtype="f32", residual=False, train=True),
        # a small head's features
        dict(name="dropout_small_f32", op="dropout", rows=100, cols=784, dtype="f32", rate=0.5, residual=False),
        # the branch of a residual block over a training batch
        dict(name="dropout_residual_batch", op="dropout", rows=16384, cols=4096, dtype="bf16", rate=0.1, residual=True),
        # a handful of prompt tokens looked up for serving
        dict(name="embed_few_tokens", op="embedding", tokens=8, vocab=32768, cols=1024, dtype="bf16", train=False),
        # a training batch on an odd vocabulary, gradient of the whole table
        dict(name="embed_train", op="embedding", tokens=16384, vocab=50001, cols=1024, dtype="bf16", train=True),
        # a long batch on a large vocabulary in full precision
        dict(name="embed_train_large_f32", op="embedding", tokens=65536, vocab=131072, cols=1024, dtype="f32", train=True),
        # a classifier's evaluation batch: forward only
        dict(name="xent_eval_classes", op="vocab_xent", tokens=100, vocab=1000, cols=2048, dtype="bf16", bias=True, train=False),
        # full precision training step with odd sizes
        dict(name="xent_train_odd_f32", op="vocab_xent", tokens=777, vocab=10007, cols=512, dtype="f32", bias=True, train=True),
        # ordinary bf16 training step, ragged token count and vocabulary
        dict(name="xent_train_ragged", op="vocab_xent", tokens=4093, vocab=50001, cols=1024, dtype="bf16", bias=False, train=True),
        # the head of a wide model over a large vocabulary
        dict(name="xent_train_large", op="vocab_xent", tokens=8192, vocab=131072, cols=4096, dtype="bf16", bias=False, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("layer_norm", "dropout", "embedding", "vocab_xent"))
    dtype = rng.choice(("bf16", "f32"))
    if op in ("layer_norm", "dropout"):
        cols = _log_int(rng, 16, 16384)
        if rng.random() < 0.5:
            cols = cols // 8 * 8
        rows = _log_int(rng, 1, max(1, min(16384, (32 if op == "layer_norm" else 64) * 2 ** 20 // cols)))
        case = dict(op=op, rows=rows, cols=cols, dtype=dtype, residual=rng.random() < 0.5)
        if op == "dropout":
            return dict(case, rate=rng.choice((0.0, 0.1, 0.25, 0.5, 0.9)))
        return dict(case, train=rng.random() < 0.7)
    cols = _log_int(rng, 8, 4096)
    if rng.random() < 0.7:
        cols = max(8, cols // 8 * 8)
    if op == "embedding":
        vocab = _log_int(rng, 64, min(131072, 2 ** 27 // cols))
        return dict(op=op, tokens=_log_int(rng, 1, min(65536, 2 ** 26 // cols)), vocab=vocab, cols=cols, dtype=dtype,
                    train=rng.random() < 0.7)
    vocab = _log_int(rng, 2, 131072)
    most = 8192 if dtype == "bf16" else max(1, min(8192, 2 ** 37 // (vocab * cols)))
    return dict(op=op, tokens=_log_int(rng, 1, most), vocab=vocab, cols=cols, dtype=dtype, bias=rng.random() < 0.5,
                train=rng.random() < 0.7)


# ----------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)

    s = {"case": case}
    if case["op"] == "layer_norm":
        r, c = case["rows"], case["cols"]
        s["x"] = normal(r, c, std=1.5, mean=0.25)
        s["residual"] = normal(r, c) if case["residual"] else None
        s["weight"] = normal(c, std=0.1, mean=1.0, dtype=torch.float32)      # parameters stay in full precision
        s["bias"] = normal(c, std=0.1, dtype=torch.float32)
        if case["train"]:
            s["dy"] = normal(r, c)
            s["dh"] = normal(r, c) if case["residual"] else None            # gradient of the residual stream itself
    elif case["op"] == "dropout":
        r, c = case["rows"], case["cols"]
        s["x"], s["dy"] = normal(r, c), normal(r, c)
        s["residual"] = normal(r, c) if case["residual"] else None
        s["seed"], s["step"] = 0x9D2C5680 * (int(seed) + 1) % 2 ** 63, int(seed) % 100003
    elif case["op"] == "embedding":
        n, v, c = case["tokens"], case["vocab"], case["cols"]
        # token frequencies fall with the index like 1 / k
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        s["ids"] = (torch.exp(u * math.log(v + 1.0)) - 1.0).long().clamp_(0, v - 1)
        s["table"] = normal(v, c, std=0.02)
        if case["train"]:
            s["dy"] = normal(n, c)
    else:
        n, v, c = case["tokens"], case["vocab"], case["cols"]
        s["weight"] = normal(v, c, std=2.0 / math.sqrt(c))
        s["bias"] = normal(v, std=0.1, dtype=torch.float32) if case["bias"] else None
        labels = torch.randint(0, v, (n,), generator=g, device="cuda")
        # half of the rows know their answer by a wide margin, a tenth is padding
        knows = torch.rand(n, generator=g, device="cuda") < 0.5
        knows[0] = False
        w = s["weight"].index_select(0, labels).float()
        pull = w / w.norm(dim=1, keepdim=True).clamp_min(1e-6) * (10.0 + 0.5 * math.sqrt(c))
        s["features"] = (torch.randn((n, c), generator=g, device="cuda") + torch.where(knows[:, None], pull, 0.0)).to(dt)
        pad = torch.rand(n, generator=g, device="cuda") < 0.1
        pad[0] = False
        s["labels"] = torch.where(pad, IGNORE, labels)
    return s


# -------------------------------------------------------------------------------------------------------- own calls
def _run_own(s):
    case, op = s["case"], s["case"]["op"]
    if op == "layer_norm":
        from distributed_tensorflow_amd.ops.layernorm import layer_norm_bwd, layer_norm_fwd
        r = layer_norm_fwd(s["x"], s["weight"], s["bias"], EPS, residual=s["residual"])
        out = {"y": r.y}
        if case["residual"]:
            out["h"] = r.h
        if case["train"]:
            out["dx"], out["dw"], out["db"] = layer_norm_bwd(s["dy"], r, s["weight"], dh=s["dh"])
        return out
    if op == "dropout":
        from distributed_tensorflow_amd.ops.dropout import dropout_apply
        return {"y": dropout_apply(s["x"], case["rate"], s["seed"], s["step"], residual=s["residual"]),
                "dx": dropout_apply(s["dy"], case["rate"], s["seed"], s["step"])}
    if op == "embedding":
        from distributed_tensorflow_amd.ops.embedding import embedding_bwd, embedding_fwd
        scale = math.sqrt(case["cols"])
        out = {"y": embedding_fwd(s["ids"], s["table"], scale)}
        if case["train"]:
            out["dtable"] = embedding_bwd(s["dy"], s["ids"], case["vocab"], scale)
        return out
    from distributed_tensorflow_amd.ops.vocab_xent import vocab_xent_bwd, vocab_xent_fwd
    r = vocab_xent_fwd(s["features"], s["weight"], s["labels"], s["bias"], ignore_index=IGNORE)
    out = {"loss": r.loss, "loss_rows": r.loss_rows, "hits": r.hits}
    if case["train"]:
        d = vocab_xent_bwd(r, s["features"], s["weight"], s["labels"], s["bias"])
        out["dfeatures"], out["dweight"] = d[0], d[1]
        if case["bias"]:
            out["dbias"] = d[2]
    return out


# ------------------------------------------------------------------------------------------------------ plain forms
def _philox_words(n_blocks, seed, step, device):
    """Philox4x32-10 (Salmon et al., 2011): the four words of counter blocks (i, step) under the key ``seed``."""
    m32 = 0xFFFFFFFF
    i = torch.arange(n_blocks, device=device, dtype=torch.int64)
    c0, c1 = i & m32, i >> 32
    c2, c3 = torch.full_like(i, step & m32), torch.full_like(i, (step >> 32) & m32)
    k0, k1 = seed & m32, (seed >> 32) & m32
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57                 # 64-bit products; the sign bit is only a bit here
        c0, c1, c2, c3 = ((p1 >> 32) & m32) ^ c1 ^ k0, p1 & m32, ((p0 >> 32) & m32) ^ c3 ^ k1, p0 & m32
        k0, k1 = (k0 + 0x9E3779B9) & m32, (k1 + 0xBB67AE85) & m32
    return c0, c1, c2, c3


def _keep_mask(n, rate, seed, step, device):
    """Element i is kept iff the i % 8-th 16-bit piece of counter block i // 8 is at least round(rate * 65536)."""
    words = torch.stack(_philox_words(-(-n // 8), seed, step, device), 1)
    pieces = torch.stack((words & 0xFFFF, words >> 16), 2).reshape(-1)[:n]
    return pieces >= int(round(rate * 65536))


def _drop_scale(rate):
    return 65536.0 / (65536 - int(round(rate * 65536)))


def _run_plain(s):
    case, op = s["case"], s["case"]["op"]
    dt = _DTYPES[case["dtype"]]
    if op == "layer_norm":
        h = s["x"]
        if case["residual"]:
            h = (h.float() + s["residual"].float()).to(dt)       # the stream is stored in its own type
        x = h.float()
        centred = x - x.mean(1, keepdim=True)
        rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)
        xhat = centred * rstd
        out = {"y": (xhat * s["weight"] + s["bias"]).to(dt)}
        if case["residual"]:
            out["h"] = h
        if case["train"]:
            dy = s["dy"].float()
            gw = dy * s["weight"]
            dx = rstd * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))
            if case["residual"]:
                dx = dx + s["dh"].float()
            out["dx"], out["dw"], out["db"] = dx.to(dt), (dy * xhat).sum(0), dy.sum(0)
        return out
    if op == "dropout":
        x, dy = s["x"].float(), s["dy"].float()
        factor = _keep_mask(x.numel(), case["rate"], s["seed"], s["step"], x.device).view_as(x) * _drop_scale(case["rate"])
        y = x * factor
        if case["residual"]:
            y = y + s["residual"].float()
        return {"y": y.to(dt), "dx": (dy * factor).to(dt)}
    if op == "embedding":
        scale = math.sqrt(case["cols"])
        out = {"y": (s["table"].index_select(0, s["ids"]).float() * scale).to(dt)}
        if case["train"]:
            grad = torch.zeros((case["vocab"], case["cols"]), device="cuda", dtype=torch.float32)
            grad.index_add_(0, s["ids"], s["dy"].float())
            out["dtable"] = (grad * scale).to(dt)
        return out
    x, w, labels = s["features"].float(), s["weight"].float(), s["labels"]
    z = x @ w.t()
    if case["bias"]:
        z = z + s["bias"]
    valid = labels != IGNORE
    lab = torch.where(valid, labels, 0)
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    target = z.gather(1, lab[:, None])
    rows = torch.where(valid, (torch.log(total) + top - target)[:, 0], 0.0)
    count = valid.sum()
    out = {"loss": rows.sum() / count, "loss_rows": rows, "hits": ((z.argmax(1) == lab) & valid).sum()}
    if case["train"]:
        del z
        dz = e.mul_((valid / count)[:, None] / total)
        dz.scatter_add_(1, lab[:, None], -(valid / count)[:, None])
        out["dfeatures"], out["dweight"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
        if case["bias"]:
            out["dbias"] = dz.sum(0)
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ----------------------------------------------------------------------------------------------------- 64-bit values
def _mul32(a, b):
    """High and low 32 bits of the product of 32-bit values, by 16-bit limbs."""
    al, ah, bl, bh = a & 0xFFFF, a >> 16, b & 0xFFFF, b >> 16
    low, mid1, mid2 = al * bl, ah * bl, al * bh
    carry = (low >> 16) + (mid1 & 0xFFFF) + (mid2 & 0xFFFF)
    return ah * bh + (mid1 >> 16) + (mid2 >> 16) + (carry >> 16), ((carry & 0xFFFF) << 16) | (low & 0xFFFF)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "layer_norm":
        x = s["x"].double()
        if case["residual"]:
            x = (x + s["residual"].double()).to(_DTYPES[case["dtype"]]).double()
        n = x.shape[1]
        mean = x.sum(1, keepdim=True) / n
        var = ((x - mean) ** 2).sum(1, keepdim=True) / n
        xhat = (x - mean) / torch.sqrt(var + EPS)
        out = {"y": xhat * s["weight"].double() + s["bias"].double()}
        if case["residual"]:
            out["h"] = x
        if case["train"]:
            dy = s["dy"].double()
            gw = dy * s["weight"].double()
            inner = n * gw - gw.sum(1, keepdim=True) - xhat * (gw * xhat).sum(1, keepdim=True)
            dx = inner / (n * torch.sqrt(var + EPS))
            out["dx"] = dx + s["dh"].double() if case["residual"] else dx
            out["dw"], out["db"] = (dy * xhat).sum(0), dy.sum(0)
        return out
    if op == "dropout":
        n, m32 = s["x"].numel(), 0xFFFFFFFF
        block = torch.arange(n, device="cuda") // 8
        c = [block & m32, block >> 32, torch.full_like(block, s["step"] & m32), torch.full_like(block, s["step"] >> 32)]
        key = [s["seed"] & m32, s["seed"] >> 32]
        for _ in range(10):
            h0, l0 = _mul32(c[0], 0xD2511F53)
            h1, l1 = _mul32(c[2], 0xCD9E8D57)
            c = [h1 ^ c[1] ^ key[0], l1, h0 ^ c[3] ^ key[1], l0]
            key = [(key[0] + 0x9E3779B9) & m32, (key[1] + 0xBB67AE85) & m32]
        lane = torch.arange(n, device="cuda") % 8
        word = torch.where(lane < 2, c[0], torch.where(lane < 4, c[1], torch.where(lane < 6, c[2], c[3])))
        bits = torch.where(lane % 2 == 0, word % 65536, word // 65536)
        drop = int(round(case["rate"] * 65536))
        factor = ((bits >= drop).double() * (65536.0 / (65536 - drop))).view_as(s["x"])
        y = s["x"].double() * factor
        return {"y": y + s["residual"].double() if case["residual"] else y, "dx": s["dy"].double() * factor}
    if op == "embedding":
        scale = math.sqrt(case["cols"])
        out = {"y": s["table"].double()[s["ids"]] * scale}
        if case["train"]:
            order = torch.argsort(s["ids"], stable=True)
            runs = torch.bincount(s["ids"], minlength=case["vocab"])
            sums = torch.cat([torch.zeros((1, case["cols"]), device="cuda", dtype=torch.float64),
                              s["dy"].double()[order].cumsum(0)])
            end = runs.cumsum(0)
            out["dtable"] = (sums[end] - sums[end - runs]) * scale
        return out
    x, w, labels = s["features"].double(), s["weight"].double(), s["labels"]
    z = torch.matmul(x, w.t())
    if case["bias"]:
        z += s["bias"].double()
    valid = labels != IGNORE
    count = valid.sum().double()
    rows = torch.arange(z.shape[0], device="cuda")
    lab = labels.clamp_min(0)
    hits = (valid & (z.argmax(1) == lab)).sum()
    lse = torch.logsumexp(z, 1)
    loss = torch.where(valid, lse - z[rows, lab], 0.0)
    out = {"loss": loss.sum() / count, "loss_rows": loss, "hits": hits}
    if case["train"]:
        dz = z.sub_(lse[:, None]).exp_()
        dz[rows, lab] -= 1.0
        dz *= (valid.double() / count)[:, None]
        out["dfeatures"], out["dweight"] = torch.matmul(dz, w), torch.matmul(dz.t(), x)
        if case["bias"]:
            out["dbias"] = dz.sum(0)
    return out


# ---------------------------------------------------------------------------------------------------------- the work
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] in ("layer_norm", "dropout"):
        n, c = case["rows"] * case["cols"], case["cols"]
        if case["op"] == "dropout":                              # x, dy [, residual] in, y, dx out
            return {"bytes": n * e * (5 if case["residual"] else 4), "flops": 4 * n}
        tensors = (4 if case["residual"] else 2) + ((3 if case["residual"] else 2) if case["train"] else 0)
        return {"bytes": n * e * tensors + 4 * c * (4 if case["train"] else 2), "flops": n * (24 if case["train"] else 8)}
    if case["op"] == "embedding":
        n, v, c = case["tokens"], case["vocab"], case["cols"]
        used = min(n, v)
        if not case["train"]:
            return {"bytes": 8 * n + (n + used) * c * e, "flops": n * c}
        return {"bytes": 8 * n + (2 * n + used + v) * c * e, "flops": 3 * n * c}
    n, v, c = case["tokens"], case["vocab"], case["cols"]
    operands = (n + v) * c * e + 8 * n + (4 * v if case["bias"] else 0)
    return {"bytes": operands * (2 if case["train"] else 1), "flops": (6 if case["train"] else 2) * n * v * c}
