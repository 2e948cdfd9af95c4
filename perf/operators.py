"""The operators around the FFN projections, as cases that can be measured: the root-mean-square norm with the residual's
addition and 8-bit outputs, the dense Q8_0 projection of 8-bit activations, and the low-rank adapters of many requests
beside a shared projection.

``own = False`` computes each operator in its plain form from elementary torch operations, ``own = True`` through the
library's entry points. Activations are F32 [token][feature], weights in the types that a GGUF stores.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-6


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of a Mistral-7B decode step: the norm before the FFN, for SeedDelta tensors (F32) and dense ones (8 bit)
        {"name": "norm-decode", "op": "norm", "tokens": 1, "n": 4096, "res": True, "f32": True, "q8": True},
        # a batch of decoding requests on Gemma-3 1B, the first norm of a layer (no residual yet), F32 only
        {"name": "norm-batch", "op": "norm", "tokens": 37, "n": 1152, "res": False, "f32": True, "q8": False},
        # a long prompt through the norm of a layer whose tensors are all dense
        {"name": "norm-prompt", "op": "norm", "tokens": 8192, "n": 4096, "res": True, "f32": False, "q8": True},
        # one token through a Mistral-7B gate that has no payload and stays dense
        {"name": "dense-decode", "op": "dense", "tokens": 1, "n_in": 4096, "n_out": 14336},
        # a ragged batch of requests through its down projection
        {"name": "dense-batch", "op": "dense", "tokens": 11, "n_in": 14336, "n_out": 4096},
        # one ubatch of a prompt on Gemma-3 4B
        {"name": "dense-ubatch", "op": "dense", "tokens": 512, "n_in": 2560, "n_out": 10240},
        # four ubatches at once on Mistral-7B
        {"name": "dense-prompt", "op": "dense", "tokens": 2048, "n_in": 4096, "n_out": 14336},
        # one request with an adapter on a Mistral-7B gate
        {"name": "lora-decode", "op": "lora", "tokens": 1, "n_in": 4096, "n_out": 14336, "adapters": 8, "rank": 16, "mixed": False, "type": "f16", "order": "each"},
        # 48 decoding requests over 32 adapters of three ranks
        {"name": "lora-batch", "op": "lora", "tokens": 48, "n_in": 4096, "n_out": 14336, "adapters": 32, "rank": 32, "mixed": True, "type": "f16", "order": "each"},
        # one ubatch of three requests' prompts on a down projection, adapters as trained (F32)
        {"name": "lora-ubatch", "op": "lora", "tokens": 512, "n_in": 14336, "n_out": 4096, "adapters": 3, "rank": 64, "mixed": False, "type": "f32", "order": "runs"},
        # long prompts of four requests, some of them without an adapter
        {"name": "lora-prompt", "op": "lora", "tokens": 4096, "n_in": 4096, "n_out": 14336, "adapters": 4, "rank": 16, "mixed": False, "type": "f16", "order": "runs"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "dense", "lora"])
    if op == "norm":
        q8 = rng.random() < 0.5
        n = _log(rng, 1024, 16384)
        n = n // 32 * 32 if q8 else n
        return {"op": op, "tokens": min(_log(rng, 1, 8192), 8192 * 4096 // n), "n": n, "res": rng.random() < 0.7, "f32": not q8 or rng.random() < 0.5, "q8": q8}
    if op == "dense":
        n_in, n_out = _log(rng, 1024, 14336) // 32 * 32, _log(rng, 1024, 14336)
        return {"op": op, "tokens": min(_log(rng, 1, 2048), 2048 * 4096 * 14336 // (n_in * n_out)), "n_in": n_in, "n_out": n_out}
    n_in, n_out = _log(rng, 1024, 14336), _log(rng, 1024, 14336)
    tokens = min(_log(rng, 1, 4096), 4096 * (4096 + 14336) // (n_in + n_out))
    return {"op": op, "tokens": tokens, "n_in": n_in, "n_out": n_out, "adapters": _log(rng, 1, 32), "rank": _log(rng, 4, 64) if tokens <= 1024 else _log(rng, 4, 16),
            "mixed": rng.random() < 0.5, "type": rng.choice(["f16", "f32"]), "order": rng.choice(["each", "runs"])}


def _ranks(case):
    return [max(1, case["rank"] >> (a % 3)) if case["mixed"] else case["rank"] for a in range(case["adapters"])]


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _inputs(case, seed):
    """What the operator's formula reads, on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    T = case["tokens"]
    if case["op"] == "norm":
        n = case["n"]
        x = rand(T, n) * (1.0 + 9.0 * (torch.rand(n, generator=g, device="cuda") < 0.01))    # a residual stream has a few large channels
        return {"x": x, "res": 0.5 * rand(T, n) if case["res"] else None, "weight": 1.0 + 0.2 * rand(n)}
    n_in, n_out = case["n_in"], case["n_out"]
    if case["op"] == "dense":
        w, x = 0.02 * rand(n_out, n_in // 32, 32), rand(T, n_in // 32, 32)
        dw, dx = (w.abs().amax(2) / 127).half(), x.abs().amax(2) / 127
        return {"wq": torch.round(w / dw.float()[:, :, None]).clamp(-127, 127).to(torch.int8), "wd": dw,
                "xq": torch.round(x / dx[:, :, None]).clamp(-127, 127).to(torch.int8), "xd": dx}
    R, nA, ranks = case["rank"], case["adapters"], torch.tensor(_ranks(case), device="cuda")
    t = torch.float16 if case["type"] == "f16" else torch.float32
    live = torch.arange(R, device="cuda") < ranks[:, None]
    if case["order"] == "each":
        ids = torch.randint(0, nA, (T,), generator=g, device="cuda")
    else:
        cut = torch.rand(T, generator=g, device="cuda").argsort()[: nA - 1].sort().values
        ids = torch.bucketize(torch.arange(T, device="cuda"), cut, right=True).clamp(max=nA - 1)
    none = torch.rand(nA, generator=g, device="cuda") < 0.1
    ids = torch.where(none[ids], -1, ids) if T > 1 else ids
    return {"x": rand(T, n_in), "base": rand(T, n_out), "ids": ids.to(torch.int32), "scale": 0.5 + torch.rand(nA, generator=g, device="cuda"),
            "a": (rand(nA, R, n_in) / math.sqrt(n_in) * live[:, :, None]).to(t), "b": (0.3 * rand(nA, n_out, R) * live[:, None, :]).to(t)}


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    if own:
        import llama_cpp_amd  # noqa: F401
        from llama_cpp_amd import scan, seeddelta, sublayer
        seeddelta.init(torch.cuda.current_device())
        T = case["tokens"]
        s["lib"] = sublayer
        if case["op"] == "norm":
            n = case["n"]
            s["sum"] = torch.empty_like(s["x"]) if case["res"] else None
            s["y"] = torch.empty_like(s["x"]) if case["f32"] else None
            if case["q8"]:
                s["q"], s["d"] = torch.empty(T, n, dtype=torch.int8, device="cuda"), torch.empty(T, n // 32, device="cuda")
        elif case["op"] == "dense":
            raw = torch.cat([s["wd"][:, :, None].view(torch.uint8), s["wq"].view(torch.uint8)], 2).reshape(case["n_out"], -1)
            s["handle"], s["y"] = scan.DenseWeight(raw.cpu().numpy()), torch.empty(T, case["n_out"], device="cuda")
        else:
            a, b, ranks = s["a"].cpu().numpy(), s["b"].cpu().numpy(), _ranks(case)
            s["handle"] = sublayer.LoraSet([(np.ascontiguousarray(a[i, :r]), np.ascontiguousarray(b[i, :, :r]), float(v)) for i, (r, v) in enumerate(zip(ranks, s["scale"].tolist()))])
            s["y"] = torch.empty_like(s["base"])
            s["ws"] = torch.empty(s["handle"].workspace_bytes(T), dtype=torch.uint8, device="cuda")
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------
def _own(s):
    c, lib, st = s["case"], s["lib"], torch.cuda.current_stream().cuda_stream
    T = c["tokens"]
    p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    if c["op"] == "norm":
        n = c["n"]
        q8 = lib.Q8View(s["q"].data_ptr(), n, s["d"].data_ptr(), n // 32) if c["q8"] else None
        lib.rms_norm_device(p(s["x"]), n, n, T, weight_ptr=p(s["weight"]), eps=EPS, res_ptr=p(s["res"]), ldr=n, sum_ptr=p(s["sum"]), lds=n, y_ptr=p(s["y"]), ldy=n, q8=q8, stream=st)
        values = torch.mul(s["q"].view(T, -1, 32), s["d"][:, :, None]).view(T, n) if c["q8"] else None     # what the 8 bits stand for
        return {"sum": s["sum"], "y": s["y"], "values": values}
    if c["op"] == "dense":
        n_in, n_out = c["n_in"], c["n_out"]
        lib.dense_forward_q8_device(s["handle"], lib.Q8View(s["xq"].data_ptr(), n_in, s["xd"].data_ptr(), n_in // 32), T, s["y"].data_ptr(), n_out, stream=st)
        return {"y": s["y"]}
    s["handle"].apply_device(p(s["ids"]), p(s["x"]), c["n_in"], T, p(s["y"]), c["n_out"], base_ptr=p(s["base"]), ldb=c["n_out"], ws_ptr=p(s["ws"]), ws_bytes=s["ws"].numel(), stream=st)
    return {"y": s["y"]}


def run(s):
    if own:
        return _own(s)
    c = s["case"]
    if c["op"] == "norm":
        x = s["x"] + s["res"] if c["res"] else s["x"]
        if not c["q8"]:
            y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * s["weight"]
            return {"sum": x if c["res"] else None, "y": y, "values": None}
        # in 64 bits: a value next to the border of two 8-bit steps goes to the right one
        z = x.double()
        z = z / torch.sqrt((z * z).mean(1, keepdim=True) + EPS) * s["weight"]
        blocks = z.view(c["tokens"], -1, 32)
        amax = blocks.abs().amax(2, keepdim=True)
        values = torch.round(blocks * (127.0 / amax)).float() * (amax / 127.0).float()
        return {"sum": x if c["res"] else None, "y": z.float() if c["f32"] else None, "values": values.view(c["tokens"], -1)}
    if c["op"] == "dense":
        w = (s["wq"].float() * s["wd"].float()[:, :, None]).view(c["n_out"], -1)
        x = (s["xq"].float() * s["xd"][:, :, None]).view(c["tokens"], -1)
        return {"y": x @ w.t()}
    nA, R = c["adapters"], c["rank"]
    # the rank-R images under every adapter, kept where the token has that adapter
    u = (s["x"] @ s["a"].float().view(nA * R, -1).t()).view(-1, nA, R)
    mine = (s["ids"][:, None] == torch.arange(nA, device="cuda", dtype=torch.int32)).float() * s["scale"]
    return {"y": s["base"] + (u * mine[:, :, None]).view(-1, nA * R) @ s["b"].float().transpose(1, 2).reshape(nA * R, -1)}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    T = case["tokens"]
    if case["op"] == "norm":
        n = case["n"]
        per = 4 + 8 * case["res"] + 4 * case["f32"] + (1 + 4 / 32) * case["q8"]
        return {"bytes": T * n * per + 4 * n, "flops": 6 * T * n}
    n_in, n_out = case["n_in"], case["n_out"]
    if case["op"] == "dense":
        return {"bytes": n_out * n_in * 34 / 32 + T * n_in * 36 / 32 + 4 * T * n_out, "flops": 2 * T * n_in * n_out}
    ranks = _ranks(case)
    mean = sum(ranks) / len(ranks)
    return {"bytes": 4 * T * (n_in + 2 * n_out + 1) + min(T, len(ranks)) * mean * (n_in + n_out) * (2 if case["type"] == "f16" else 4), "flops": 2 * T * mean * (n_in + n_out)}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    d = {k: v.double() for k, v in s.items() if v is not None and k != "ids"}
    T = case["tokens"]
    if case["op"] == "norm":
        total = d["x"] if s["res"] is None else (s["x"] + s["res"]).double()       # the sum is F32 by definition: the next layer reads it
        y = d["weight"] * total * torch.pow(total.pow(2).sum(1, keepdim=True).div(case["n"]).add(EPS), -0.5)
        values = None
        if case["q8"]:
            step = y.view(T, -1, 32).abs().max(2, keepdim=True).values / 127
            values = (torch.round(y.view(T, -1, 32) / step) * step).reshape(T, -1)
        return {"sum": None if s["res"] is None else d["x"] + d["res"], "y": y if case["f32"] else None, "values": values}
    if case["op"] == "dense":
        return {"y": torch.mm((d["xq"] * d["xd"].unsqueeze(2)).flatten(1), (d["wq"] * d["wd"].unsqueeze(2)).flatten(1).t().contiguous())}
    y = d["base"].clone()
    for k in range(case["adapters"]):
        at = (s["ids"] == k).nonzero()[:, 0]
        y[at] += d["scale"][k] * torch.mm(torch.mm(d["x"][at], d["a"][k].t().contiguous()), d["b"][k].t().contiguous())
    return {"y": y}
