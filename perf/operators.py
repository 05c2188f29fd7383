"""What the operators of 8-bit decoders and of scoring are measured by: products in 8-bit integers, the norms around a block, and the log
probabilities of tokens.

``listed()`` holds the cases, ``draw(rng)`` gives more of the same ranges.  ``own`` chooses between the operators' plain form (elementary torch
operations) and the calls a user of the framework makes.

  linear    y = (sum_k q[t, k] w[n, k]) s[t] c[n] (+ bias) (+ residual), or silu(gate) * up of it over a weight whose rows are blocks of 128 gate
            and 128 up rows.  w is int8 with one factor c a channel, laid out beforehand; x comes in a float type and is turned into 8 bits within
            the call: s[t] = max |x[t]| / 127, q = round(127 x / max |x[t]|), halves to even.
  norm      x' = a x + b g post(y), h = pre(x'), both RMS norms, g one value a channel or the sigmoid of one a token and channel.
  handover  the norm, its rows in 8 bits, and the product that takes them.
  logprobs  of a given token: log probability, entropy of its row, how many tokens are more likely, and the ``top`` likeliest with theirs.

Sizes are those of the decoders the framework has presets for (hidden 896, 2048, 3584, feed-forward 4864, 18944, vocabularies 151936 and 152064),
and odd ones.
"""
import math

import torch

own = False

EPS = 1e-6
NEG = float("-inf")
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _linear(name, m, n, k, dtype="bf16", bias=False, residual=False, gated=False):
    return {"name": name, "kind": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias, "residual": residual, "gated": gated}


def _norm(name, m, k, stream="bf16", dtype="bf16", post=True, gate="none", n=0):
    return {"name": name, "kind": "norm" if n == 0 else "handover", "m": m, "k": k, "n": n, "stream": stream, "dtype": dtype, "post": post, "gate": gate}


def _logprobs(name, rows, vocab, dtype="bf16", top=0, entropy=False, masked=False):
    return {"name": name, "kind": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top, "entropy": entropy, "masked": masked}


def listed():
    return [
        # one user's next token: the attention's input projection, where latency counts
        _linear("linear_one", 1, 4608, 3584, bias=True),
        # a batch of users: the feed-forward's way back onto the residual stream, bound by the weights
        _linear("linear_batch", 64, 3584, 18944, residual=True),
        # a short question's gated feed-forward
        _linear("linear_gated_short", 77, 37888, 3584, gated=True),
        # a prompt through a projection whose sizes divide nothing
        _linear("linear_ragged", 1333, 1001, 2039, dtype="f16", bias=True),
        # long prompts together: the largest product, bound by the tensor cores
        _linear("linear_prompts", 8192, 3584, 18944, residual=True),
        # one token between two blocks, norms on both sides
        _norm("norm_one", 1, 3584, gate="channel"),
        # long prompts with a 32-bit residual stream and a gate for each token
        _norm("norm_prompts", 8192, 3584, stream="f32", gate="token"),
        # a batch's rows handed to an 8-bit projection
        _norm("handover_batch", 256, 2048, n=5120),
        # one generated token with its alternatives, as a chat with log probabilities asks for
        _logprobs("logprobs_one", 1, 151936, top=5, entropy=True),
        # a batch with the most alternatives that a request may have
        _logprobs("logprobs_batch", 256, 152064, top=20, entropy=True),
        # rows behind a grammar's mask, in 32 bits: most of the vocabulary is gone, of some rows all of it
        _logprobs("logprobs_masked", 33, 50257, dtype="f32", top=8, entropy=True, masked=True),
        # scoring documents: every position's own token
        _logprobs("logprobs_score", 3500, 152064),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "gated", "norm", "handover", "logprobs", "logprobs"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "linear":
        m, n, k = _log(rng, 1, 8192), _log(rng, 33, 18944), _log(rng, 65, 18944)
        while m * n * k > 8192 * 3584 * 18944:
            m //= 2
        c = _linear("", m, n, k, dtype, bias=rng.random() < 0.5, residual=rng.random() < 0.5)
    elif kind == "gated":
        c = _linear("", _log(rng, 1, 3000), 256 * _log(rng, 3, 148), _log(rng, 65, 4096), dtype, gated=True)
    elif kind == "norm":
        c = _norm("", _log(rng, 1, 8192), _log(rng, 65, 8192), rng.choice(("bf16", "f32")), dtype, rng.random() < 0.7, rng.choice(("none", "channel", "token")))
    elif kind == "handover":
        c = _norm("", _log(rng, 1, 2048), _log(rng, 65, 8192), rng.choice(("bf16", "f32")), "bf16", rng.random() < 0.7, rng.choice(("none", "channel", "token")),
                  n=_log(rng, 65, 8192))
    else:
        vocab = rng.choice((32000, 50257, 151936, 152064, _log(rng, 100, 200000)))
        rows = _log(rng, 1, 3000)
        c = _logprobs("", rows, vocab, dtype if rows * vocab < 1e8 else "bf16", rng.choice((0, 0, 1, 5, 20)), rng.random() < 0.5, rng.random() < 0.3)
    del c["name"]
    return c


def _int8_weight(n, k, g):
    """Rows begin at multiples of 16 bytes, as a program lays its weights out when it loads them."""
    w = torch.randint(-90, 91, (n, (k + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)[:, :k]
    return w, (0.5 + torch.rand(n, generator=g, device="cuda")) * (0.02 / 52.0)


def _activations(m, k, g):
    """Channels of different sizes, as a decoder's hidden states have them."""
    return torch.randn(m, k, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(k, generator=g, device="cuda"))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
    s = {"case": case}
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.empty(rows, vocab, dtype=TYPES[case["dtype"]], device="cuda")
        for r in range(0, rows, 256):
            x[r:r + 256] = 2.5 * rand(min(256, rows - r), vocab)
        tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        # a model that is sure of itself puts one token far above the rest
        at = torch.arange(rows, device="cuda")
        x[at, tokens.long()] += (12.0 * torch.rand(rows, generator=g, device="cuda")).to(x.dtype)
        if case["masked"]:
            keep = torch.rand(rows, 1, generator=g, device="cuda") ** 8
            x.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") > keep, NEG)
            x[rows // 2] = NEG
        return s | {"logits": x, "tokens": tokens}
    m, k, n = case["m"], case["k"], case["n"]
    t = TYPES[case["dtype"]]
    if case["kind"] == "linear":
        s["x"] = _activations(m, k, g).to(t)
        s["w"], s["c"] = _int8_weight(n, k, g)
        s["bias"] = rand(n) if case["bias"] else None
        s["residual"] = rand(m, n).to(t) if case["residual"] else None
        return s
    s["x"] = (4.0 * _activations(m, k, g)).to(TYPES[case["stream"]])
    s["y"] = _activations(m, k, g).to(t)
    s["post"] = 1.0 + 0.2 * rand(k) if case["post"] else None
    s["pre"] = 1.0 + 0.2 * rand(k)
    s["gate"] = {"none": lambda: None, "channel": lambda: 1.0 + 0.3 * rand(k), "token": lambda: rand(m, k).to(t)}[case["gate"]]()
    s["x_out"] = torch.empty_like(s["x"])
    if n:
        s["w"], s["c"] = _int8_weight(n, k, g)
    return s


# what the stream and the block's output are weighed by
X_SCALE, Y_SCALE = 1.0, 0.7


# ---- the plain form ----
def _rows(x):
    """Rows in 8 bits: whole numbers as floats, and their factors.  The quotient is taken in 64 bits: it decides on which side of a half it lies."""
    peak = x.abs().amax(1, keepdim=True)
    q = torch.round(x.double() * 127.0 / torch.where(peak > 0, peak, 1.0).double()).float()
    return q, peak / 127.0


def _product(q, s, w, c):
    # whole numbers below 2^24 all the way: exact in 32 bits
    return (q @ w.float().t()) * s * c


def _rms(x, w):
    return x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * w


def _plain_linear(s):
    case, x = s["case"], s["x"]
    q, f = _rows(x.float())
    y = _product(q, f, s["w"], s["c"])
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["gated"]:
        y = y.view(y.shape[0], -1, 2, 128)
        gate, up = y[:, :, 0], y[:, :, 1]
        y = (gate / (1.0 + torch.exp(-gate)) * up).reshape(y.shape[0], -1)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(x.dtype)


def _plain_stream(s):
    y = s["y"].float()
    if s["post"] is not None:
        y = _rms(y, s["post"])
    if s["gate"] is not None:
        y = y * (s["gate"] if s["gate"].dim() == 1 else torch.sigmoid(s["gate"].float()))
    return X_SCALE * s["x"].float() + Y_SCALE * y


def _plain_norm(s):
    x = _plain_stream(s)
    return {"x": x.to(s["x"].dtype), "h": _rms(x, s["pre"]).to(s["y"].dtype)}


def _plain_handover(s):
    x = _plain_stream(s)
    q, f = _rows(_rms(x, s["pre"]))
    return {"x": x.to(s["x"].dtype), "y": _product(q, f, s["w"], s["c"]).to(s["y"].dtype)}


def _plain_logprobs(s):
    case, x = s["case"], s["logits"].float()
    vocab, at = case["vocab"], s["tokens"].long().unsqueeze(1)
    peak = x.amax(1, keepdim=True)
    d = x - peak
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    given = x.gather(1, at)
    out = {"logprob": (given - peak - torch.log(z)).squeeze(1), "rank": (x > given).sum(1).int()}
    if case["entropy"]:
        # what has no weight adds nothing; a row without any is not a number
        out["entropy"] = (torch.log(z) - torch.where(e == 0, 0.0, e * d).sum(1, keepdim=True) / z).squeeze(1)
    if case["top"]:
        # the value in the order of whole numbers, then the lower index
        bits = x.view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * vocab + torch.arange(vocab - 1, -1, -1, device=x.device)
        ids = vocab - 1 - torch.topk(key, case["top"], dim=1).values.remainder(vocab)
        out["top_ids"] = ids.int()
        out["top_logprobs"] = x.gather(1, ids) - peak - torch.log(z)
    return out


# ---- the framework's calls ----
def _own(s):
    from onnx_genai_b200 import ops
    from onnx_genai_b200.ops import int8

    case = s["case"]
    if case["kind"] == "linear":
        return int8.gemm_int8(s["x"], s["w"], s["c"], bias=s["bias"], residual=s["residual"], epilogue="swiglu" if case["gated"] else "none")
    if case["kind"] == "logprobs":
        r = ops.token_logprobs(s["logits"], s["tokens"], top=case["top"], entropy=case["entropy"])
        out = {"logprob": r.logprob, "rank": r.rank}
        if case["entropy"]:
            out["entropy"] = r.entropy
        if case["top"]:
            out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        return out
    handover = case["kind"] == "handover"
    h = int8.block_norm(s["x"], s["y"], post=s["post"], gate=s["gate"], pre=s["pre"], eps=EPS, x_scale=X_SCALE, y_scale=Y_SCALE,
                        gate_sigmoid=case["gate"] == "token", x_out=s["x_out"], int8=handover, out_dtype=None if handover else s["y"].dtype)
    if not handover:
        return {"x": s["x_out"], "h": h}
    return {"x": s["x_out"], "y": int8.gemm_int8(h, s["w"], s["c"], out_dtype=s["y"].dtype)}


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "norm": _plain_norm, "handover": _plain_handover, "logprobs": _plain_logprobs}[state["case"]["kind"]](state)


def work(case):
    size = lambda t: TYPES[t].itemsize    # noqa: E731
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size(case["dtype"]) + case["rows"] * (16 + 8 * case["top"]), "flops": 4.0 * n}
    m, n, k = case["m"], case["n"], case["k"]
    e = size(case["dtype"])
    if case["kind"] == "linear":
        out = n // 2 if case["gated"] else n
        return {"bytes": m * k * e + n * k + 4 * n + m * out * e * (2 if case["residual"] else 1), "flops": 2.0 * m * n * k}
    stream = 2 * m * k * size(case["stream"]) + m * k * e * (2 if case["gate"] == "token" else 1) + 4 * k * (2 if case["post"] else 1)
    if case["kind"] == "norm":
        return {"bytes": stream + m * k * e, "flops": 10.0 * m * k}
    return {"bytes": stream + n * k + 4 * n + m * n * e, "flops": 2.0 * m * n * k + 10.0 * m * k}


# ---- 64 bits, from the definitions ----
def _exact_rows(x):
    peak = x.abs().max(dim=1, keepdim=True).values
    ratio = x * 127.0 / peak.clamp_min(1e-300)
    return ratio.round(), peak / 127.0


def _exact_dense(q, s, w, c):
    """A block of weight rows at a time: their 64-bit copies are large."""
    parts = [(q @ w[i:i + 4096].double().T) for i in range(0, w.shape[0], 4096)]
    return torch.cat(parts, 1) * s * c.double().unsqueeze(0)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        cols = {"logprob": [], "entropy": [], "top_logprobs": []}
        for r in range(0, case["rows"], 256):
            lp = torch.log_softmax(s["logits"][r:r + 256].double(), -1)
            cols["logprob"].append(lp.gather(1, s["tokens"][r:r + 256, None].long())[:, 0])
            if case["entropy"]:
                cols["entropy"].append(torch.special.entr(lp.exp()).sum(-1))
            if case["top"]:
                cols["top_logprobs"].append(lp.sort(-1, descending=True).values[:, :case["top"]])
        out = {k: torch.cat(v) for k, v in cols.items() if v}
        return out | {"rank": None} | ({"top_ids": None} if case["top"] else {})
    if case["kind"] == "linear":
        y = _exact_dense(*_exact_rows(s["x"].double()), s["w"], s["c"])
        if case["bias"]:
            y += s["bias"].double()
        if case["gated"]:
            blocks = y.unflatten(1, (-1, 256))
            y = (torch.nn.functional.silu(blocks[..., :128]) * blocks[..., 128:]).flatten(1)
        if case["residual"]:
            y += s["residual"].double()
        return y
    y = s["y"].double()
    if case["post"]:
        y = y / (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["post"].double()
    if case["gate"] == "channel":
        y = y * s["gate"].double()
    elif case["gate"] == "token":
        y = y / (1.0 + (-s["gate"].double()).exp())
    x = X_SCALE * s["x"].double() + Y_SCALE * y
    h = x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * s["pre"].double()
    if case["kind"] == "norm":
        return {"x": x, "h": h}
    return {"x": x, "y": _exact_dense(*_exact_rows(h), s["w"], s["c"])}
