"""Measured cases of the token-model operators: embedding rows and their gradient, layer norm forward and
backward, log probabilities of given tokens with entropy and top alternatives and their gradient, and the
orthogonalised update of a weight matrix.

`own` chooses between the plain form (elementary torch operations in 32 bits) and the calls a user makes of
neuzephyr_b200. The cases stand for one step of training or serving a token model on one GPU.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7
LN_EPS = 1e-5


def listed():
    return [
        # the tokens of one decoding step of a batch of requests: nothing but latency
        {"name": "embed_step", "op": "embed", "tokens": 32, "vocab": 32768, "dim": 2048, "dtype": "f16", "index": "i32", "zipf": True},
        # the tokens of a training batch or of a long prompt
        {"name": "embed_batch", "op": "embed", "tokens": 16384, "vocab": 131072, "dim": 5120, "dtype": "bf16", "index": "i64", "zipf": True},
        # gradient of an fp32 table from 16-bit upstream gradients; a few tokens make up much of the text,
        # and a part of the batch is padding
        {"name": "embed_grad", "op": "embed_grad", "tokens": 16384, "vocab": 65536, "dim": 2048, "dtype": "bf16", "index": "i64", "zipf": True},
        # a decoding step's rows, in this framework's own type
        {"name": "norm_step", "op": "norm", "rows": 64, "dim": 1024, "dtype": "f32"},
        # a training batch with rows of an odd length: no row but the first starts on a vector's boundary
        {"name": "norm_odd", "op": "norm", "rows": 8191, "dim": 5003, "dtype": "f16"},
        # the same of a model with wide rows, backward, with the reduction of both parameters' gradients
        {"name": "norm_grad", "op": "norm_grad", "rows": 16384, "dim": 4096, "dtype": "bf16"},
        # log probabilities of the tokens of one decoding step, with alternatives: few rows, a long axis
        {"name": "logprob_step", "op": "logprob", "rows": 4, "vocab": 131072, "dtype": "bf16", "index": "i64", "top_k": 8, "scale": 1.25},
        # scoring a prompt: many rows, an odd vocabulary, fp32 logits
        {"name": "logprob_prompt", "op": "logprob", "rows": 4096, "vocab": 50021, "dtype": "f32", "index": "i64", "top_k": 5, "scale": 1.0},
        # the loss's gradient over a training batch, with an entropy term
        {"name": "logprob_grad", "op": "logprob_grad", "rows": 4096, "vocab": 131072, "dtype": "bf16", "index": "i64", "scale": 1.0},
        # a small layer's weight
        {"name": "ortho_small", "op": "ortho", "batch": 1, "rows": 256, "cols": 512, "dtype": "f32"},
        # several layers' weights of one shape, sides that are no multiple of a tile
        {"name": "ortho_batch", "op": "ortho", "batch": 4, "rows": 1000, "cols": 1400, "dtype": "bf16"},
        # a large layer's weight, taller than wide
        {"name": "ortho_large", "op": "ortho", "batch": 1, "rows": 8192, "cols": 4096, "dtype": "f32"},
    ]


def _spread(rng, lo, hi):
    """An integer spread over the logarithm of lo..hi; half of them odd, the others with the factors of two sizes have."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and v > 64:
        step = 64 if v > 512 else 8
        v = v // step * step
    else:
        v |= 1
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "norm", "norm_grad", "logprob", "logprob_grad", "ortho"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    index = rng.choice(["i32", "i64"])
    if op in ("embed", "embed_grad"):
        dim = _spread(rng, 64, 8192)
        vocab = _spread(rng, 1000, min(131072, (1 << 27) // dim))
        return {"op": op, "tokens": _spread(rng, 1, min(32768, (1 << 26) // dim)), "vocab": vocab, "dim": dim, "dtype": dtype,
                "index": index, "zipf": rng.random() < 0.7}
    if op in ("norm", "norm_grad"):
        dim = _spread(rng, 64, 16384)
        return {"op": op, "rows": _spread(rng, 1, min(65536, (1 << 25) // dim)), "dim": dim, "dtype": dtype}
    if op in ("logprob", "logprob_grad"):
        vocab = _spread(rng, 1000, 200000)
        case = {"op": op, "rows": _spread(rng, 1, min(16384, (1 << 27) // vocab)), "vocab": vocab, "dtype": dtype, "index": index,
                "scale": rng.choice([1.0, 0.7, 1.25])}
        if op == "logprob":
            case["top_k"] = rng.choice([0, 1, 4, 8, 20])
        return case
    rows, cols = _spread(rng, 128, 4096), _spread(rng, 128, 8192)
    if rng.random() < 0.5:
        rows, cols = cols, rows
    short = min(rows, cols)
    batch = max(1, min(rng.choice([1, 1, 2, 6]), (1 << 33) // (short * rows * cols)))
    return {"op": "ortho", "batch": batch, "rows": rows, "cols": cols, "dtype": dtype}


# ---- inputs ----------------------------------------------------------------------------------------------
def _token_probabilities(vocab, device):
    p = 1.0 / (torch.arange(vocab, device=device, dtype=torch.float64) + 2.7)
    return p / p.sum()


def _tokens(case, count, vocab, gen, device):
    """Token numbers: by Zipf's law with the frequent ones spread over the vocabulary, or uniform."""
    if case.get("zipf"):
        cum = torch.cumsum(_token_probabilities(vocab, device), 0)
        rank = torch.searchsorted(cum, torch.rand(count, device=device, dtype=torch.float64, generator=gen)).clamp_(max=vocab - 1)
        tokens = (rank * 7919 + 13) % vocab
    else:
        tokens = torch.randint(0, vocab, (count,), device=device, generator=gen)
    return tokens.to(torch.int32 if case["index"] == "i32" else torch.int64)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    s = dict(case)
    op, dtype = case["op"], DTYPES[case["dtype"]]

    def normal(*shape, to=dtype, std=1.0, mean=0.0):
        return torch.randn(*shape, device=device, generator=gen).mul_(std).add_(mean).to(to)

    if op == "embed":
        s["table"] = normal(case["vocab"], case["dim"], std=0.02)
        s["tokens"] = _tokens(case, case["tokens"], case["vocab"], gen, device)
        s["scale"] = math.sqrt(case["dim"])
    elif op == "embed_grad":
        s["tokens"] = _tokens(case, case["tokens"], case["vocab"], gen, device)
        s["padding"] = case["vocab"] // 2
        s["tokens"][: case["tokens"] // 16] = s["padding"]  # rows of short sequences filled up
        s["dy"] = normal(case["tokens"], case["dim"], std=1e-2)
        s["scale"] = math.sqrt(case["dim"])
        s["dtable"] = torch.empty(case["vocab"], case["dim"], device=device)  # the gradient buffer a program keeps
    elif op in ("norm", "norm_grad"):
        x = torch.randn(case["rows"], case["dim"], device=device, generator=gen)
        x *= torch.rand(case["rows"], 1, device=device, generator=gen) * 3 + 0.2
        x += torch.randn(case["rows"], 1, device=device, generator=gen)
        s["x"] = x.to(dtype)
        s["gamma"] = normal(case["dim"], to=torch.float32, std=0.2, mean=1.0)
        s["beta"] = normal(case["dim"], to=torch.float32, std=0.2)
        if op == "norm_grad":
            xf = s["x"].double()  # what the forward pass kept
            mean = xf.mean(1)
            s["mean"] = mean.float()
            s["rstd"] = ((xf - mean[:, None]).square().mean(1) + LN_EPS).rsqrt().float()
            s["dy"] = normal(case["rows"], case["dim"], std=1e-2)
            s["dx"] = torch.empty(case["rows"], case["dim"], device=device, dtype=dtype)
            s["dgamma"] = torch.empty(case["dim"], device=device)
            s["dbeta"] = torch.empty(case["dim"], device=device)
    elif op in ("logprob", "logprob_grad"):
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.randn(rows, vocab, device=device, generator=gen)
        logits *= torch.rand(rows, 1, device=device, generator=gen) * 3 + 0.5
        s["targets"] = _tokens({"index": case["index"], "zipf": True}, rows, vocab - vocab // 50, gen, device)
        # the model favours the token that follows, and the vocabulary's last columns stand for no token
        logits.scatter_add_(1, s["targets"].long()[:, None], torch.rand(rows, 1, device=device, generator=gen) * 12)
        logits[:, vocab - vocab // 50:] = -math.inf
        s["logits"] = logits.to(dtype)
        if op == "logprob_grad":
            s["targets"][: rows // 16] = -100  # positions without a target
            s["dlogprob"] = torch.full((rows,), -1.0 / rows, device=device)
            s["dentropy"] = torch.full((rows,), -0.01 / rows, device=device)
            lse, ent = [], []
            for part in s["logits"].split(256):  # what the forward pass kept
                z = part.double() * case["scale"]
                lse.append(torch.logsumexp(z, 1))
                p = torch.exp(z - lse[-1][:, None])
                ent.append(-torch.where(p > 0, p * (z - lse[-1][:, None]), 0.0).sum(1))
            s["lse"], s["entropy"] = torch.cat(lse).float(), torch.cat(ent).float()
            s["dlogits"] = torch.empty_like(s["logits"])
    else:
        # a gradient is a sum over tokens of products of features whose sizes fall off
        b, rows, cols = case["batch"], case["rows"], case["cols"]
        tokens = 2 * max(rows, cols)
        up = torch.randn(b, rows, tokens, device=device, generator=gen)
        up *= (torch.arange(rows, device=device) + 1.0).pow(-0.5)[:, None]
        act = torch.randn(b, tokens, cols, device=device, generator=gen)
        act *= (torch.arange(cols, device=device) + 1.0).pow(-0.5)
        s["g"] = torch.matmul(up, act).mul_(1e-4).to(dtype)
    return s


# ---- one pass --------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    import neuzephyr_b200 as nz
    op = s["op"]
    if op == "embed":
        return nz.embedding(s["table"], s["tokens"], scale=s["scale"])
    if op == "embed_grad":
        return nz.embedding_backward(s["dy"], s["tokens"], s["dtable"], scale=s["scale"], padding_index=s["padding"], overwrite=True)
    if op == "norm":
        return nz.layernorm_forward(s["x"], s["gamma"], s["beta"], eps=LN_EPS)
    if op == "norm_grad":
        nz.layernorm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"], dx=s["dx"], dgamma=s["dgamma"], dbeta=s["dbeta"],
                              overwrite_dx=True, overwrite_dparams=True)
        return s["dx"], s["dgamma"], s["dbeta"]
    if op == "logprob":
        r = nz.token_logprobs(s["logits"], s["targets"], scale=s["scale"], top_k=s["top_k"])
        return {"logprob": r.logprob, "entropy": r.entropy, "lse": r.lse, "top_logprob": r.top_logprob, "top_index": r.top_index}
    if op == "logprob_grad":
        return nz.token_logprobs_backward(s["logits"], s["targets"], s["lse"], s["entropy"], s["dlogprob"], s["dentropy"],
                                          scale=s["scale"], out=s["dlogits"])
    return nz.orthogonalize(s["g"], steps=NS_STEPS, coefficients=NS_COEFFICIENTS, eps=NS_EPS, out_dtype=torch.bfloat16)


def _run_plain(s):
    op = s["op"]
    if op == "embed":
        return (s["table"][s["tokens"].long()].float() * s["scale"]).to(s["table"].dtype)
    if op == "embed_grad":
        dy = s["dy"].float() * torch.where(s["tokens"] == s["padding"], 0.0, s["scale"])[:, None]
        return torch.zeros(s["vocab"], s["dim"], device=dy.device).index_add_(0, s["tokens"].long(), dy)
    if op == "norm":
        x = s["x"].float()
        mean = x.mean(1)
        centred = x - mean[:, None]
        rstd = torch.rsqrt(centred.square().mean(1) + LN_EPS)
        return (centred * rstd[:, None] * s["gamma"] + s["beta"]).to(s["x"].dtype), mean, rstd
    if op == "norm_grad":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        xhat = (s["x"].float() - s["mean"][:, None]) * rstd
        g = dy * s["gamma"]
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        return dx.to(s["x"].dtype), (dy * xhat).sum(0), dy.sum(0)
    if op == "logprob":
        return _logprob_plain(s)
    if op == "logprob_grad":
        logq = s["logits"].float() * s["scale"] - s["lse"][:, None]
        p = torch.exp(logq)
        t = s["targets"].long()
        inside = (t >= 0) & (t < s["vocab"])
        dl = torch.where(inside, s["dlogprob"], 0.0)
        d = -dl[:, None] * p - torch.where(p > 0, s["dentropy"][:, None] * p * (logq + s["entropy"][:, None]), 0.0)
        d.scatter_add_(1, torch.where(inside, t, 0)[:, None], dl[:, None])
        return (d * s["scale"]).to(s["logits"].dtype)
    return _ortho_plain(s["g"])


def _logprob_plain(s):
    x, t = s["logits"].float(), s["targets"].long()
    z = x * s["scale"]
    top = z.amax(1, keepdim=True)
    z = z - top
    e = torch.exp(z)
    total = e.sum(1)
    log_total = torch.log(total)
    inside = (t >= 0) & (t < s["vocab"])
    picked = z.gather(1, torch.where(inside, t, 0)[:, None])[:, 0]
    out = {"logprob": torch.where(inside, picked - log_total, 0.0),
           "entropy": log_total - torch.where(e > 0, e * z, 0.0).sum(1) / total,
           "lse": top[:, 0] + log_total}
    # ranks by value, then by the lower token: one whole number for both
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
    key = key * (1 << 32) + (s["vocab"] - torch.arange(s["vocab"], device=x.device))
    at = s["vocab"] - (key.topk(s["top_k"], dim=1, sorted=True)[0] & 0xFFFFFFFF)
    out["top_logprob"] = z.gather(1, at) - log_total[:, None]
    out["top_index"] = at.to(s["targets"].dtype)
    return out


def _ortho_plain(g):
    a, b, c = NS_COEFFICIENTS
    x = g.float()
    tall = g.shape[1] > g.shape[2]
    if tall:
        x = x.transpose(1, 2)
    x = x / (torch.sqrt(x.square().sum((1, 2), keepdim=True)) + NS_EPS)
    for _ in range(NS_STEPS):
        gram = torch.matmul(x, x.transpose(1, 2))
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return (x.transpose(1, 2) if tall else x).to(torch.bfloat16).contiguous()


# ---- what a pass cannot do without -------------------------------------------------------------------------
def _rows_touched(case):
    """Expected number of different tokens."""
    n, vocab = case["tokens"], case["vocab"]
    p = _token_probabilities(vocab, "cpu") if case["zipf"] else torch.full((vocab,), 1.0 / vocab, dtype=torch.float64)
    return float((1 - torch.exp(n * torch.log1p(-p))).sum())


def work(case):
    op, size = case["op"], SIZE[case["dtype"]]
    index = {"i32": 4, "i64": 8}[case.get("index", "i64")]
    if op == "embed":
        n, dim = case["tokens"], case["dim"]
        return {"bytes": n * index + (n + _rows_touched(case)) * dim * size, "flops": n * dim}
    if op == "embed_grad":
        n, dim = case["tokens"], case["dim"]
        return {"bytes": n * index + n * dim * size + case["vocab"] * dim * 4, "flops": 2 * n * dim}
    if op == "norm":
        n = case["rows"] * case["dim"]
        return {"bytes": 2 * n * size + 8 * case["dim"] + 8 * case["rows"], "flops": 8 * n}
    if op == "norm_grad":
        n = case["rows"] * case["dim"]
        return {"bytes": 3 * n * size + 12 * case["dim"] + 8 * case["rows"], "flops": 14 * n}
    if op == "logprob":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (index + 12 + case["top_k"] * (4 + index)), "flops": 6 * n}
    if op == "logprob_grad":
        n = case["rows"] * case["vocab"]
        return {"bytes": 2 * n * size + case["rows"] * (index + 16), "flops": 7 * n}
    m, n = sorted((case["rows"], case["cols"]))
    # both products of a matrix with its own transpose give symmetric results: half of each has to be computed
    flops = NS_STEPS * (m * m * n + m * m * m + 2 * m * m * n)
    return {"bytes": case["batch"] * m * n * (size + 2), "flops": case["batch"] * flops}


# ---- the definition in 64 bits -----------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "embed":
        return torch.index_select(s["table"], 0, s["tokens"].to(torch.int64)).double().mul_(s["scale"])
    if op == "embed_grad":
        order = torch.argsort(s["tokens"].to(torch.int64), stable=True)
        tokens = s["tokens"].to(torch.int64)[order]
        order, tokens = order[tokens != s["padding"]], tokens[tokens != s["padding"]]
        out = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device="cuda")
        seen, counts = torch.unique_consecutive(tokens, return_counts=True)
        if seen.numel():
            out[seen] = torch.segment_reduce(s["dy"][order].double() * s["scale"], "sum", lengths=counts, axis=0)
        return out
    if op == "norm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, 1, correction=0)
        r = 1.0 / torch.sqrt(var + LN_EPS)
        return torch.addcmul(s["beta"].double(), (x - mean.unsqueeze(1)) * r.unsqueeze(1), s["gamma"].double()), mean, r
    if op == "norm_grad":
        x, dy = s["x"].double(), s["dy"].double()
        mean, r = s["mean"].double().unsqueeze(1), s["rstd"].double().unsqueeze(1)
        h, g, n = (x - mean) * r, dy * s["gamma"].double(), case["dim"]
        inner = torch.einsum("rd,rd->r", g, h).unsqueeze(1) / n
        return (g - g.sum(1, keepdim=True) / n - h * inner) * r, torch.einsum("rd,rd->d", dy, h), dy.sum(0)
    if op == "logprob":
        parts = []
        for x, t in zip(s["logits"].split(256), s["targets"].split(256)):
            logq = torch.log_softmax(x.double() * case["scale"], 1)
            q = torch.exp(logq)
            ent = torch.special.entr(q).sum(1)
            lse = torch.logsumexp(x.double() * case["scale"], 1)
            parts.append((logq.gather(1, t.to(torch.int64).unsqueeze(1)).squeeze(1), ent, lse, torch.topk(logq, case["top_k"], 1)[0]))
        logp, ent, lse, top = (torch.cat(v) for v in zip(*parts))
        return {"logprob": logp, "entropy": ent, "lse": lse, "top_logprob": top, "top_index": None}
    if op == "logprob_grad":
        out = torch.empty(case["rows"], case["vocab"], dtype=torch.float64, device="cuda")
        for i in range(0, case["rows"], 256):
            j = slice(i, i + 256)
            logq = s["logits"][j].double() * case["scale"] - s["lse"][j].double().unsqueeze(1)
            q, t = torch.exp(logq), s["targets"][j].to(torch.int64)
            hit = torch.zeros_like(q)
            at = torch.nonzero(t >= 0).squeeze(1)
            hit[at, t[at]] = 1.0
            has = (t >= 0).double().unsqueeze(1)
            wave = torch.nan_to_num(q * (logq + s["entropy"][j].double().unsqueeze(1)), nan=0.0)
            out[j] = case["scale"] * (s["dlogprob"][j].double().unsqueeze(1) * has * (hit - q) - s["dentropy"][j].double().unsqueeze(1) * wave)
        return out
    a, b, c = NS_COEFFICIENTS
    out = []
    for g in s["g"].double():
        wide = g if g.shape[0] <= g.shape[1] else g.mT
        x = wide / (torch.linalg.norm(wide) + NS_EPS)
        eye = torch.eye(x.shape[0], dtype=torch.float64, device="cuda")
        for _ in range(NS_STEPS):
            gram = x @ x.mT
            x = (a * eye + gram @ (b * eye + c * gram)) @ x
        out.append(x if g.shape[0] <= g.shape[1] else x.mT)
    return torch.stack(out)
