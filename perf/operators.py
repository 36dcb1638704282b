"""Operators of the 8-bit rollout step: linear layers in 8-bit integers with a scale per token and per
output channel (alone, behind RMSNorm and behind SwiGLU), and sampling with temperature, top-k, top-p
and min-p from given random numbers.

``own`` selects the side: False runs the plain forms below, True the framework's operators. Formulas:

* rows to 8 bits:  a = max |x|,  s = a / 127,  q = round_half_even(127 x / a)  (a row of zeros: q = 0)
* linear:          y = s_x[t] s_w[n] sum_k q_x[t, k] q_w[n, k]  (+ bias[n]) (+ residual[t, n])
* sampling:        z = x / T;  tokens in order (value descending, index ascending); kept are the first
                   top_k of them with exp(z - z_max) >= min_p, of these the ones whose preceding share
                   of the kept mass is below top_p; the token is the first one whose cumulative mass
                   exceeds u times the mass kept. Its log-probability is that of softmax(x).
"""

import math

import torch

own = False


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _linear(name, pre, m, k, n, dtype="bfloat16", bias=False, residual=False):
    case = {"name": name} if name else {}
    return {**case, "kind": "linear", "pre": pre, "m": m, "k": k, "n": n, "dtype": dtype, "bias": bias,
            "residual": residual}


def _sample(name, rows, v, dtype="bfloat16", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False,
            masked=0.0):
    case = {"name": name} if name else {}
    return {**case, "kind": "sample", "rows": rows, "v": v, "dtype": dtype, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed, "masked": masked}


def listed():
    return [
        # one sequence decodes: the qkv projection of the 1.5B shape (latency)
        _linear("linear_1x1536x2048", "none", 1, 1536, 2048, bias=True),
        # a usual decode batch: the gate|up projection of the 1.5B shape (streams the weight)
        _linear("linear_64x1536x17920", "none", 64, 1536, 17920),
        # sizes that fit no tile, in fp16
        _linear("linear_333x1001x1111_fp16", "none", 333, 1001, 1111, dtype="float16", bias=True, residual=True),
        # a full prefill step of the engine (8192 tokens), gate|up of the 1.5B shape
        _linear("linear_8192x1536x17920", "none", 8192, 1536, 17920),
        # the LM head of the 1.5B shape on a decode batch
        _linear("linear_128x1536x151936", "none", 128, 1536, 151936),
        # input norm + qkv of the 1.5B shape on a decode batch
        _linear("rmsnorm_linear_64x1536x2048", "rmsnorm", 64, 1536, 2048, bias=True),
        # post-attention norm + gate|up of the 8B shape on a prefill chunk
        _linear("rmsnorm_linear_2048x4096x24576", "rmsnorm", 2048, 4096, 24576),
        # SwiGLU + down of the 1.5B shape on the largest usual decode batch
        _linear("swiglu_linear_256x8960x1536", "swiglu", 256, 8960, 1536, residual=True),
        # the same on a full prefill step
        _linear("swiglu_linear_8192x8960x1536", "swiglu", 8192, 8960, 1536, residual=True),
        # one row with every filter (latency)
        _sample("sample_1x151936_filters", 1, 151936, temperature=0.8, top_k=50, top_p=0.95, min_p=0.02),
        # the engine's largest usual batch, every row with settings of its own, a tenth of the entries masked
        _sample("sample_256x151936_mixed", 256, 151936, mixed=True, masked=0.1),
        # plain sampling at temperature 1 of an odd, smaller vocabulary in fp16
        _sample("sample_100x32003_fp16", 100, 32003, dtype="float16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.65:
        pre = rng.choice(["none", "rmsnorm", "swiglu"])
        m = _log_int(rng, 1, 8192)
        k = _log_int(rng, 96, 8960)
        if rng.random() < 0.5:
            k = max(64, k // 64 * 64)
        if pre != "none":
            k = max(8, k // 8 * 8)  # hidden and intermediate sizes of the framework's norm and SwiGLU
        n = _log_int(rng, 96, 17920)
        if rng.random() < 0.5:
            n = max(64, n // 64 * 64)
        while m * k * n > 8192 * 1536 * 17920:
            m = max(1, m // 2)
        return _linear(None, pre, m, k, n, rng.choice(["bfloat16", "bfloat16", "float16"]) if pre == "none"
                       else "bfloat16", rng.random() < 0.4, rng.random() < 0.4)
    v = _log_int(rng, 1000, 152064)
    rows = min(_log_int(rng, 1, 256), 256 * 151936 // v)
    mixed = rng.random() < 0.5
    return _sample(None, rows, v, rng.choice(["bfloat16", "bfloat16", "float16"]),
                   round(rng.uniform(0.3, 1.5), 3), rng.choice([0, 1, 20, 50, 1000]),
                   rng.choice([1.0, round(rng.uniform(0.5, 0.99), 3)]),
                   rng.choice([0.0, round(rng.uniform(0.001, 0.2), 4)]), mixed, rng.choice([0.0, 0.1, 0.9]))


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    """The case's tensors, from the seed alone (activations with a few large channels and tokens, as the
    residual stream has them; peaked logits)."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = getattr(torch, case["dtype"])

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    s = {}
    if case["kind"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        if case["pre"] == "swiglu":
            s["x"] = randn(m, 2 * k).to(dt)
        else:
            x = randn(m, k) * (1.0 + 8.0 * (rand(k) < 0.01)) * (0.25 + 2.0 * rand(m, 1))
            s["x"] = x.to(dt)
        if case["pre"] == "rmsnorm":
            s["norm_w"] = (1.0 + 0.1 * randn(k)).to(dt)
        s["w"] = (randn(n, k) * (0.02 * (0.5 + rand(n, 1)))).to(dt)
        s["bias"] = (0.1 * randn(n)).to(dt) if case["bias"] else None
        s["residual"] = randn(m, n).to(dt) if case["residual"] else None
        return s
    rows, v = case["rows"], case["v"]
    x = 2.0 * randn(rows, v)
    peaks = torch.randint(0, v, (rows, 48), generator=g, device=dev)
    x.scatter_add_(1, peaks, -4.0 * torch.log(rand(rows, 48).clamp_min(1e-6)))
    if case["masked"] > 0:
        x.masked_fill_(rand(rows, v) < case["masked"], float("-inf"))
        x[:, v // 2] = 3.0  # never an empty row
    s["logits"] = x.to(dt)
    s["u"] = rand(rows)
    if case["mixed"]:
        def choose(options):
            pick = torch.randint(0, len(options), (rows,), generator=g, device=dev)
            return torch.tensor(options, device=dev)[pick]

        s["temperature"] = choose([0.0, 0.6, 0.8, 1.0, 1.2])
        s["top_k"] = choose([0, 0, 20, 50, 1000]).to(torch.int32)
        s["top_p"] = choose([1.0, 0.8, 0.9, 0.95])
        s["min_p"] = choose([0.0, 0.0, 0.05, 0.1])
    else:
        s["temperature"] = torch.full((rows,), case["temperature"], device=dev)
        s["top_k"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device=dev) if case["top_k"] else None
        s["top_p"] = torch.full((rows,), case["top_p"], device=dev) if case["top_p"] < 1.0 else None
        s["min_p"] = torch.full((rows,), case["min_p"], device=dev) if case["min_p"] > 0.0 else None
    return s


EPS = 1e-6  # of the RMSNorm


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["kind"] == "linear":
        # the weight in 8 bits is laid out once, when the weights are loaded
        w = s.pop("w")
        if own:
            from accerl_agent_b200 import ops

            s["w8"] = ops.quantize_rows(w)
        else:
            s["w8"] = _quantize(w.float())
    return s


# ------------------------------------------------------------------------------------------------
# the plain forms
# ------------------------------------------------------------------------------------------------
def _quantize(x):
    a = x.abs().amax(1, keepdim=True)
    # the quotient decides between neighbouring whole numbers: in 64 bits
    q = torch.round(127.0 * x.double() / a.double()).nan_to_num_(0.0)
    return q, (a / 127.0)


def _plain_linear(s):
    case = s["case"]
    dt = getattr(torch, case["dtype"])
    x = s["x"]
    if case["pre"] == "rmsnorm":
        xf = x.float()
        y = xf * torch.rsqrt((xf * xf).mean(1, keepdim=True) + EPS)
        # the framework's norm rounds before and after the weight
        xf = (y.to(dt).float() * s["norm_w"].float()).to(dt).float()
    elif case["pre"] == "swiglu":
        k = case["k"]
        gate, up = x[:, :k].float(), x[:, k:].float()
        xf = ((gate / (1.0 + torch.exp(-gate))).to(dt).float() * up).to(dt).float()
    else:
        xf = x.float()
    q, sx = _quantize(xf)
    wq, sw = s["w8"]
    acc = q @ wq.t()  # whole numbers beyond 24 bits: in 64 bits
    y = acc.float() * (sx * sw.t())
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(dt)


def _plain_sample(s):
    x = s["logits"].double()  # mass next to a border decides the token: in 64 bits
    rows, v = x.shape
    x = torch.where(torch.isnan(x), float("-inf"), x)
    top = x.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    xs, order = torch.sort(x, dim=1, descending=True, stable=True)
    t = s["temperature"].double().unsqueeze(1)
    w = torch.where(t > 0, torch.exp((xs - top) / t), (xs == top).double())
    rank = torch.arange(v, device=x.device).unsqueeze(0)
    keep = torch.ones_like(w, dtype=torch.bool)
    if s["top_k"] is not None:
        k = s["top_k"].long().unsqueeze(1)
        keep &= (rank < k) | (k <= 0)
    keep &= (rank < 1) | (t > 0)
    if s["min_p"] is not None:
        keep &= (w >= s["min_p"].double().unsqueeze(1)) | (rank < 1)
    w = w * keep
    if s["top_p"] is not None:
        p = s["top_p"].double().unsqueeze(1)
        before = torch.cumsum(w, 1) - w
        w = w * ((before < p * w.sum(1, keepdim=True)) | (rank < 1) | (p >= 1))
    cum = torch.cumsum(w, 1)
    target = s["u"].double().unsqueeze(1) * cum[:, -1:]
    pos = (cum <= target).sum(1, keepdim=True).clamp_max(v - 1)
    tok = order.gather(1, pos)
    return tok.squeeze(1), (x.gather(1, tok) - lse).squeeze(1).float()


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if not own:
        return _plain_linear(state) if case["kind"] == "linear" else _plain_sample(state)
    from accerl_agent_b200 import ops

    if case["kind"] == "sample":
        return ops.sample_inverse_cdf(state["logits"], state["u"], state["temperature"], top_k=state["top_k"],
                                      top_p=state["top_p"], min_p=state["min_p"])
    if case["pre"] == "rmsnorm":
        x = ops.rmsnorm_quantize(state["x"], state["norm_w"], EPS)
    elif case["pre"] == "swiglu":
        x = ops.swiglu_quantize(state["x"])
    else:
        x = state["x"]
    return ops.linear_int8(x, state["w8"], bias=state["bias"], residual=state["residual"])


def work(case):
    """Activations, weight (8 bits and a scale per channel) and residual read once, the output written
    once; logits read once, a token and a log-probability written per row."""
    if case["kind"] == "sample":
        rows, v = case["rows"], case["v"]
        # one exponential's worth of work per logit
        return {"bytes": 2 * rows * v + 32 * rows, "flops": 4 * rows * v}
    m, k, n = case["m"], case["k"], case["n"]
    b = m * k * (4 if case["pre"] == "swiglu" else 2) + n * k + 4 * n + 2 * m * n
    if case["pre"] == "rmsnorm":
        b += 2 * k
    if case["bias"]:
        b += 2 * n
    if case["residual"]:
        b += 2 * m * n
    return {"bytes": b, "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------------
# from the definition, in 64 bits
# ------------------------------------------------------------------------------------------------
def _round_rows(x):
    """(whole numbers, step) of the rows of a 64-bit matrix: floor and its remainder instead of round."""
    step = x.abs().max(dim=1).values.div(127.0)
    r = x / torch.where(step > 0, step, torch.ones_like(step)).unsqueeze(1)
    lo = torch.floor(r)
    rest = r - lo
    up = (rest > 0.5) | ((rest == 0.5) & (torch.remainder(lo, 2.0) == 1.0))
    return lo + up.double(), step


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "linear":
        x = s["x"].double()
        if case["pre"] == "rmsnorm":
            # the norm's own two roundings are part of its definition in the framework
            dt = getattr(torch, case["dtype"])
            norm = x.pow(2).sum(1).div(case["k"]).add(EPS).sqrt()
            x = ((x / norm.unsqueeze(1)).to(dt).double() * s["norm_w"].double()).to(dt).double()
        elif case["pre"] == "swiglu":
            dt = getattr(torch, case["dtype"])
            gate, up = x.chunk(2, dim=1)
            x = ((gate * torch.sigmoid(gate)).to(dt).double() * up).to(dt).double()
        qx, sx = _round_rows(x)
        qw, sw = _round_rows(s["w"].double())
        out = torch.empty(case["m"], case["n"], dtype=torch.float64, device=x.device)
        for n0 in range(0, case["n"], 8192):
            part = torch.einsum("mk,nk->mn", qx, qw[n0 : n0 + 8192])
            out[:, n0 : n0 + 8192] = part * sx.unsqueeze(1) * sw[n0 : n0 + 8192].unsqueeze(0)
        if s["bias"] is not None:
            out += s["bias"].double()
        if s["residual"] is not None:
            out += s["residual"].double()
        return out
    tokens, logprobs = [], []
    for r in range(case["rows"]):
        x = s["logits"][r].double()
        ids = torch.nonzero(x > float("-inf")).squeeze(1)
        vals, perm = torch.sort(x[ids], descending=True, stable=True)
        ids = ids[perm]
        t = float(s["temperature"][r])
        n = ids.numel()
        if t <= 0:
            n, t = 1, 1.0
        k = int(s["top_k"][r]) if s["top_k"] is not None else 0
        if k > 0:
            n = min(n, k)
        mass = torch.exp((vals[:n] - vals[0]) / t)
        if s["min_p"] is not None:
            n = max(1, int((mass >= float(s["min_p"][r])).sum()))
            mass = mass[:n]
        p = float(s["top_p"][r]) if s["top_p"] is not None else 1.0
        if p < 1.0:
            cum = torch.cumsum(mass, 0)
            n = min(n, int(torch.searchsorted(cum, (p * cum[-1]).reshape(1), right=False)) + 1)
            mass = mass[:n]
        cum = torch.cumsum(mass, 0)
        at = int(torch.searchsorted(cum, (float(s["u"][r]) * cum[-1]).reshape(1), right=True))
        at = min(at, n - 1)
        tokens.append(ids[at])
        logprobs.append(vals[at] - torch.logsumexp(vals, 0))
    return torch.stack(tokens), torch.stack(logprobs)
