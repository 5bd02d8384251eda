"""Performance cases of the dense layers and of sampling on one MI355X.

A case is a dict of plain values; its "kind" names the operator that `run` calls.

  linear    act(W x + bias) + residual, W in BF16 or row-int8 (dense.linear)
  ffn       f(W_gate x, W_up x), f SiLU or SiTU gating; with keep also the two
            projections, which the backward pass reads (dense.gated_ffn)
  ffn_bwd   its gradients: x, W_gate and W_up (dense.gated_ffn_backward)
  sample    a token per row of logits by temperature, top-k, top-p and min-p from
            given uniform numbers (sampling.sample)

Sizes are the shared expert of the K3 block (hidden 7168, intermediate 6144), preset
2's widths (hidden 7168, intermediate 2048), and generic ones.  `run` computes the plain
form, elementary torch operations in 32 bits (64 for sampling, where a rounding can
change the token), or makes the framework's calls where `own` is true.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_MOST_FLOPS = 4.9e11     # of the largest listed case (ffn_bwd_4096)


# ------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # one decoded token through a down projection and its residual add: launch bound
        dict(name="linear_one", kind="linear", rows=7168, cols=2048, m=1, x="bf16",
             weights="bf16", act="none", bias=False, residual=True),
        # a draft batch through row-int8 weights, fp32 activations
        dict(name="linear_int8_m9", kind="linear", rows=7168, cols=6144, m=9, x="f32",
             weights="int8", act="none", bias=False, residual=True),
        # a short prompt, ragged, through a projection with bias and activation
        dict(name="linear_gelu_m333", kind="linear", rows=3584, cols=7168, m=333, x="f32",
             weights="bf16", act="gelu", bias=True, residual=False),
        # a prompt chunk through the shared expert's down projection, int8 weights
        dict(name="linear_int8_m1024", kind="linear", rows=7168, cols=6144, m=1024, x="bf16",
             weights="int8", act="none", bias=False, residual=True),
        # a long prompt or a training batch through the same projection
        dict(name="linear_m4096", kind="linear", rows=7168, cols=6144, m=4096, x="bf16",
             weights="bf16", act="none", bias=True, residual=True),
        # one decoded token through a gated block of preset 2's widths
        dict(name="ffn_one", kind="ffn", inter=2048, hidden=7168, m=1, x="bf16", act="silu",
             keep=False),
        # a prompt through the K3 shared expert's gate and up, fp32 activations
        dict(name="ffn_situ_m2048", kind="ffn", inter=6144, hidden=7168, m=2048, x="f32",
             act="situ", keep=False),
        # the forward half of a training step, projections kept
        dict(name="ffn_train_m4096", kind="ffn", inter=2048, hidden=7168, m=4096, x="bf16",
             act="silu", keep=True),
        # the backward half of the same step
        dict(name="ffn_bwd_m4096", kind="ffn_bwd", inter=2048, hidden=7168, m=4096, x="bf16",
             act="silu"),
        # a small ragged batch in fp32 through odd widths
        dict(name="ffn_bwd_f32_m517", kind="ffn_bwd", inter=1003, hidden=2050, m=517, x="f32",
             act="situ"),
        # the next token of one sequence
        dict(name="sample_one", kind="sample", m=1, vocab=131072, x="f32"),
        # a serving batch, every row with its own parameters, an odd vocabulary
        dict(name="sample_m96", kind="sample", m=96, vocab=150001, x="bf16"),
    ]


def _cost(case: dict) -> float:
    return work(case)["flops"] * (3 if case["x"] == "f32" else 1)


def draw(rng: random.Random) -> dict:
    def log_int(lo: int, hi: int, step: int = 1) -> int:
        v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
        return min(hi, max(lo, step * round(v / step)))

    x = rng.choice(("f32", "bf16"))
    kind = rng.choice(("linear", "linear", "ffn", "ffn_bwd", "sample"))
    if kind == "sample":
        return dict(kind=kind, m=log_int(1, 128), vocab=log_int(1000, 200000), x=x)
    step = rng.choice((64, 64, 8, 1))
    wide, deep = log_int(64, 12288, step), log_int(64, 8192, step)
    if kind == "linear":
        case = dict(kind=kind, rows=wide, cols=deep, m=log_int(1, 8192), x=x,
                    weights=rng.choice(("bf16", "int8")),
                    act=rng.choice(("none", "silu", "gelu")), bias=rng.random() < 0.5,
                    residual=rng.random() < 0.5)
    else:
        case = dict(kind=kind, inter=min(wide, 8192), hidden=deep,
                    m=log_int(1 if kind == "ffn" else 16, 8192), x=x,
                    act=rng.choice(("silu", "situ")))
        if kind == "ffn":
            case["keep"] = rng.random() < 0.5
    while _cost(case) > _MOST_FLOPS:
        case["m"] = case["m"] * 2 // 3
    return case


# ------------------------------------------------------------------ the inputs
def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = _DTYPES[case["x"]]

    def normal(*shape: int, scale: float = 1.0, dtype: torch.dtype = dt) -> torch.Tensor:
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def uniform(n: int, lo: float, hi: float) -> torch.Tensor:
        return torch.rand(n, generator=g, device="cuda") * (hi - lo) + lo

    st = dict(case)
    m = case["m"]
    if case["kind"] == "sample":
        v = case["vocab"]
        st["logits"] = normal(m, v, scale=2.5)
        # greedy rows among the sampled ones, small and absent top-k, top-p and min-p
        st["temperature"] = uniform(m, 0.5, 1.4) * (uniform(m, 0.0, 1.0) > 0.1)
        k = torch.exp(uniform(m, 1.0, math.log(v))).to(torch.int32)
        st["top_k"] = k * (uniform(m, 0.0, 1.0) > 0.3)
        st["top_p"] = torch.where(uniform(m, 0.0, 1.0) > 0.3, uniform(m, 0.5, 1.0),
                                  torch.ones(m, device="cuda"))
        st["min_p"] = uniform(m, 0.0, 0.1) * (uniform(m, 0.0, 1.0) > 0.5)
        st["u"] = torch.rand(m, generator=g, device="cuda")
        return st
    if case["kind"] == "linear":
        r, c = case["rows"], case["cols"]
        st["x"] = normal(m, c)
        if case["weights"] == "int8":
            st["w"] = torch.randint(-127, 128, (r, c), generator=g, device="cuda",
                                    dtype=torch.int8)
            st["s"] = uniform(r, 0.5, 1.5) / (73.0 * math.sqrt(c))
        else:
            st["w"] = normal(r, c, scale=c ** -0.5, dtype=torch.bfloat16)
            st["s"] = None
        st["b"] = normal(r, dtype=torch.float32) if case["bias"] else None
        st["r"] = normal(m, r) if case["residual"] else None
        return st
    s, h = case["inter"], case["hidden"]
    st["x"] = normal(m, h)
    st["wg"] = normal(s, h, scale=h ** -0.5, dtype=torch.bfloat16)
    st["wu"] = normal(s, h, scale=h ** -0.5, dtype=torch.bfloat16)
    if case["kind"] == "ffn_bwd":
        st["gate"], st["up"], st["dh"] = normal(m, s), normal(m, s), normal(m, s)
    return st


# ------------------------------------------------------------------ one pass
def run(st: dict):
    kind = st["kind"]
    if own:
        from deltafin_amd import dense, sampling
        if kind == "linear":
            return dense.linear(st["w"], st["x"], bias=st["b"], activation=st["act"],
                                residual=st["r"], row_scales=st["s"])
        if kind == "ffn":
            return dense.gated_ffn(st["wg"], st["wu"], st["x"], st["act"], keep=st["keep"])
        if kind == "ffn_bwd":
            return dense.gated_ffn_backward(st["wg"], st["wu"], st["x"], st["gate"], st["up"],
                                            st["dh"], st["act"])
        return sampling.sample(st["logits"], st["u"], temperature=st["temperature"],
                               top_k=st["top_k"], top_p=st["top_p"], min_p=st["min_p"])
    if kind == "sample":
        return _plain_sample(st)
    dt = st["x"].dtype
    x = st["x"].float()
    if kind == "linear":
        z = x @ st["w"].float().t()
        if st["s"] is not None:
            z = z * st["s"]
        if st["b"] is not None:
            z = z + st["b"]
        if st["act"] == "silu":
            z = z / (1.0 + torch.exp(-z))
        elif st["act"] == "gelu":
            z = 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
        if st["r"] is not None:
            z = z + st["r"].float()
        return z.to(dt)
    wg, wu = st["wg"].float(), st["wu"].float()
    if kind == "ffn":
        gate, up = x @ wg.t(), x @ wu.t()
        sig = 1.0 / (1.0 + torch.exp(-gate))
        if st["act"] == "silu":
            h = gate * sig * up
        else:
            h = 4.0 * torch.tanh(gate / 4.0) * sig * (25.0 * torch.tanh(up / 25.0))
        return (h.to(dt), gate.to(dt), up.to(dt)) if st["keep"] else h.to(dt)
    gate, up, dh = st["gate"].float(), st["up"].float(), st["dh"].float()
    sig = 1.0 / (1.0 + torch.exp(-gate))
    if st["act"] == "silu":
        dg = dh * up * sig * (1.0 + gate * (1.0 - sig))
        du = dh * gate * sig
    else:
        t, v = torch.tanh(gate / 4.0), torch.tanh(up / 25.0)
        dg = dh * ((1.0 - t * t) * sig + 4.0 * t * sig * (1.0 - sig)) * (25.0 * v)
        du = dh * (4.0 * t * sig) * (1.0 - v * v)
    dx = dg @ wg + du @ wu
    return dx.to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt)


def _plain_sample(st: dict) -> torch.Tensor:
    logits = st["logits"].double()
    m, v = logits.shape
    ordered, index = torch.sort(logits, dim=1, descending=True, stable=True)
    t = st["temperature"].double().unsqueeze(1)
    w = torch.exp((ordered - ordered[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)))
    mass = torch.cumsum(w, dim=1)
    k = st["top_k"].long().unsqueeze(1)
    k = torch.where((k <= 0) | (k > v), torch.full_like(k, v), k)
    p = st["top_p"].double().unsqueeze(1)
    n_p = 1 + (mass < p * torch.gather(mass, 1, k - 1)).sum(dim=1, keepdim=True)
    n_p = torch.where(p >= 1.0, torch.full_like(k, v), n_p)
    n_m = (w >= st["min_p"].double().unsqueeze(1)).sum(dim=1, keepdim=True)
    n = torch.minimum(torch.minimum(k, n_p), n_m)
    n = torch.where(t > 0, n, torch.ones_like(n))
    target = st["u"].double().unsqueeze(1) * torch.gather(mass, 1, n - 1)
    at = torch.minimum((mass <= target).sum(dim=1, keepdim=True), n - 1)
    return torch.gather(index, 1, at).squeeze(1).to(torch.int32)


# ------------------------------------------------------------------ its work
def work(case: dict) -> dict:
    e = 4 if case["x"] == "f32" else 2
    m = case["m"]
    if case["kind"] == "sample":
        return {"bytes": m * (case["vocab"] * e + 24), "flops": 2 * m * case["vocab"]}
    if case["kind"] == "linear":
        r, c = case["rows"], case["cols"]
        wb = r * c + 4 * r if case["weights"] == "int8" else 2 * r * c
        return {"bytes": wb + m * c * e + m * r * e * (2 if case["residual"] else 1)
                + (4 * r if case["bias"] else 0), "flops": 2 * m * r * c}
    s, h = case["inter"], case["hidden"]
    if case["kind"] == "ffn":
        return {"bytes": 4 * s * h + m * h * e + m * s * e * (3 if case["keep"] else 1),
                "flops": 4 * m * s * h}
    return {"bytes": 4 * s * h + 2 * s * h * e + 2 * m * h * e + 3 * m * s * e,
            "flops": 8 * m * s * h}


# ------------------------------------------------------------------ 64 bits
def exact(case: dict, seed: int):
    if case["kind"] == "sample":
        return None          # tokens: whole numbers
    st = prepare(case, seed)
    d = {k: v.double() for k, v in st.items() if isinstance(v, torch.Tensor)}
    if case["kind"] == "linear":
        z = torch.matmul(d["x"], d["w"].transpose(0, 1))
        z = z * d["s"] if "s" in d else z
        z = z + d["b"] if "b" in d else z
        if case["act"] == "silu":
            z = z * torch.sigmoid(z)
        elif case["act"] == "gelu":
            z = z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z + d["r"] if "r" in d else z
    g = d["gate"] if "gate" in d else torch.matmul(d["x"], d["wg"].transpose(0, 1))
    u = d["up"] if "up" in d else torch.matmul(d["x"], d["wu"].transpose(0, 1))
    sg = torch.sigmoid(g)
    if case["act"] == "silu":
        a, da = g * sg, sg + g * sg * (1 - sg)
        b, db = u, torch.ones_like(u)
    else:
        th = torch.tanh(g / 4)
        a, da = 4 * th * sg, sg / torch.cosh(g / 4) ** 2 + 4 * th * sg * (1 - sg)
        b, db = 25 * torch.tanh(u / 25), torch.cosh(u / 25) ** -2
    if case["kind"] == "ffn":
        return (a * b, g, u) if case["keep"] else a * b
    dg, du = d["dh"] * da * b, d["dh"] * a * db
    return (torch.matmul(dg, d["wg"]) + torch.matmul(du, d["wu"]),
            torch.matmul(dg.transpose(0, 1), d["x"]), torch.matmul(du.transpose(0, 1), d["x"]))
