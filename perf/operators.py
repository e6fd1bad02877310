"""The cases at which the token-step operators are measured: rotary positions, rotary with the append to
the KV cache, and sampling.

`run` computes an operator in its plain form (elementary torch operations) where `own` is false and calls the
library where it is true.  Sizes: 1536 wide activations are the LeLM's (12 heads of 128), 2200 wide the Flow
estimator's (20 heads of 110, 1000-frame windows), 16385 logits the LeLM's codebook and its end token; the others
are generic.
"""
from __future__ import annotations

import importlib.util
import math
import pathlib
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
VOCAB = 16385  # LeLM codebook of 16384 and the end token


def _ops():
    """levo2.cpp_b200/ops.py (the folder's name is not an identifier)."""
    name = "levo2_cpp_b200"
    if name not in sys.modules:
        folder = pathlib.Path(__file__).resolve().parent.parent / "levo2.cpp_b200"
        spec = importlib.util.spec_from_file_location(name, folder / "__init__.py",
                                                      submodule_search_locations=[str(folder)])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return sys.modules[name].ops


# --------------------------------------------------------------------------- cases

def _rope(name, dtype, batch, seq, q_heads, k_heads, dim, rot, layout, order="bshd", adjoint=False, scaling="none",
          start=0, magnitude=1.0):
    return {"name": name, "kind": "rope", "dtype": dtype, "batch": batch, "seq": seq, "q_heads": q_heads,
            "k_heads": k_heads, "dim": dim, "rot": rot, "interleaved": layout == "interleaved", "order": order,
            "adjoint": adjoint, "scaling": scaling, "start": start, "magnitude": magnitude}


def _append(name, dtype, batch, seq, q_heads, k_heads, dim, rot, layout, capacity, ragged=True):
    return {"name": name, "kind": "append", "dtype": dtype, "batch": batch, "seq": seq, "q_heads": q_heads,
            "k_heads": k_heads, "dim": dim, "rot": rot, "interleaved": layout == "interleaved",
            "capacity": capacity, "ragged": ragged}


def _sample(name, dtype, rows, vocab, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, spread=3.0, recent=0, ignore=0,
            per_row=False):
    return {"name": name, "kind": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "temperature": temperature,
            "top_k": top_k, "top_p": top_p, "min_p": min_p, "spread": spread, "recent": recent, "ignore": ignore,
            "per_row": per_row}


def listed():
    return [
        # one token of a guided pair (conditional and unconditional row) in the LeLM: latency
        _rope("rope one token", "f16", 2, 1, 12, 12, 128, 128, "half", start=700),
        # the LeLM's prompt of a batch of songs, q and k as they lie in a fused projection's output
        _rope("rope prompt fused qkv", "f16", 4, 2048, 12, 12, 128, 128, "half", order="qkv"),
        # a Flow window pair of the DiT: 20 heads of 110, all odd in 16-byte terms
        _rope("rope window 110", "f32", 2, 1000, 20, 20, 110, 110, "interleaved", order="bhsd"),
        # backward of a long training sequence, shared key heads, part of the head, positions far out and scaled by parts
        _rope("rope backward far", "bf16", 1, 16001, 32, 8, 128, 64, "half", adjoint=True, scaling="by_parts",
              start=100000, magnitude=1.2079),
        # a decode step of 64 requests at different lengths
        _append("append step", "bf16", 64, 1, 32, 8, 128, 128, "half", 1024),
        # ragged prompt chunks of the LeLM
        _append("append chunk ragged", "f16", 8, 1023, 12, 12, 128, 128, "interleaved", 2048),
        # the three token streams of one song: latency
        _sample("sample 3 streams top-k", "f32", 3, VOCAB, temperature=0.9, top_k=50, recent=50, ignore=16),
        # the streams of 64 songs, large k with a nucleus in it
        _sample("sample 192 streams k+p", "f32", 192, VOCAB, temperature=0.9, top_k=250, top_p=0.95, recent=50),
        # a large batch, nucleus and min-p over the whole vocabulary, settings of their own for each row
        _sample("sample 1024 rows per row", "f16", 1024, VOCAB, top_p=0.95, min_p=0.02, per_row=True),
        # one row of a large vocabulary: latency, one row over many SMs
        _sample("sample 1 row 131072", "bf16", 1, 131072, temperature=0.8, top_p=0.9),
        # flat logits (hot sampling): thousands of tokens stay in the nucleus
        _sample("sample 128 rows flat", "f32", 128, 131072, temperature=1.3, top_p=0.97, spread=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rope", "rope", "append", "sample", "sample"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    if kind == "sample":
        vocab = _log_int(rng, 33, 131072)
        rows = _log_int(rng, 1, max(1, min(1024, (1 << 24) // vocab)))
        return {k: v for k, v in _sample(
            "", dtype, rows, vocab, temperature=round(rng.uniform(0.5, 1.5), 3),
            top_k=rng.choice((0, 0, _log_int(rng, 1, 2000))), top_p=rng.choice((1.0, round(rng.uniform(0.5, 0.99), 3))),
            min_p=rng.choice((0.0, 0.0, round(rng.uniform(0.001, 0.2), 4))), spread=round(rng.uniform(0.7, 4.0), 2),
            recent=rng.choice((0, _log_int(rng, 1, 300))), ignore=rng.choice((0, 0, 16)),
            per_row=rng.random() < 0.25).items() if k != "name"}
    dim = rng.choice((64, 80, 96, 110, 128, 192, 256))
    rot = rng.choice((dim, dim, dim // 2 // 2 * 2))
    k_heads = rng.choice((1, 2, 4, 8, 12))
    q_heads = k_heads * rng.choice((1, 1, 2, 4))
    layout = rng.choice(("half", "interleaved"))
    batch = _log_int(rng, 1, 64)
    room = 300_000_000 // (2 * BYTES[dtype] * batch * (q_heads + 2 * k_heads) * dim)
    seq = _log_int(rng, 1, max(1, min(16384, room)))
    if kind == "append":
        case = _append("", dtype, batch, seq, q_heads, k_heads, dim, rot, layout,
                       seq + rng.randrange(1, 200), ragged=rng.random() < 0.7)
    else:
        case = _rope("", dtype, batch, seq, q_heads, k_heads, dim, rot, layout,
                     order=rng.choice(("bshd", "bhsd", "qkv")), adjoint=rng.random() < 0.4,
                     scaling=rng.choice(("none", "linear", "ntk", "by_parts")), start=rng.choice((0, 17, 1000003)),
                     magnitude=rng.choice((1.0, 1.2079)))
    return {k: v for k, v in case.items() if k != "name"}


def work(case):
    if case["kind"] == "sample":
        rows, n = case["rows"], case["rows"] * case["vocab"]
        small = rows * (8 + 4 + 4 + 8 * case["recent"] + (20 if case["per_row"] else 0)) + 8 * case["ignore"]
        return {"bytes": float(n * BYTES[case["dtype"]] + small), "flops": 4.0 * n}  # difference, scale, exp, sum
    tokens, e = case["batch"] * case["seq"], BYTES[case["dtype"]]
    heads = case["q_heads"] + case["k_heads"] * (2 if case["kind"] == "append" else 1)
    turned = (case["q_heads"] + case["k_heads"]) * case["rot"]
    small = 8 * tokens if case["kind"] == "rope" else 16 * case["batch"]
    return {"bytes": float(2 * tokens * heads * case["dim"] * e + small + 4 * case["rot"]),
            "flops": 3.0 * tokens * turned}


# --------------------------------------------------------------------------- inputs

def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _frequencies(rot, scaling, device):
    """Radians a position of each pair: base 10000; scaled by 8 for eight times a context of 4096."""
    base, factor, context = 10000.0, 8.0, 4096
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    theta = base ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device=device) / rot)
    if scaling == "linear":
        theta = theta / factor
    if scaling == "by_parts":  # pairs that turn often keep their pace, slow ones are stretched, a ramp between
        ramp = ((context * theta / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        theta = (1 - ramp) * theta / factor + ramp * theta
    return theta


def _normal(shape, dtype, gen):
    return torch.randn(shape, generator=gen, device=gen.device, dtype=torch.float32).to(dtype)


def prepare(case, seed):
    device = _device()
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "sample":
        return _prepare_sample(case, gen, dtype)
    b, s, hq, hk, d = case["batch"], case["seq"], case["q_heads"], case["k_heads"], case["dim"]
    state = {"case": case, "theta": _frequencies(case["rot"], case.get("scaling", "none"), device)}
    if case["kind"] == "append":
        fused = _normal((b, s, hq + 2 * hk, d), dtype, gen)  # q, k and v side by side in the projection's output
        state["q"], state["k"], state["v"] = fused[:, :, :hq], fused[:, :, hq:hq + hk], fused[:, :, hq + hk:]
        room = case["capacity"] - s
        state["lengths"] = torch.randint(0, room + 1, (b,), generator=gen, device=device)
        state["counts"] = (torch.randint(max(0, s // 4), s + 1, (b,), generator=gen, device=device)
                           if case["ragged"] else torch.full((b,), s, device=device))
        if s == 1:
            state["counts"].fill_(1)
        state["k_cache"] = torch.zeros((b, case["capacity"], hk, d), dtype=dtype, device=device)
        state["v_cache"] = torch.zeros_like(state["k_cache"])
        state["q_out"] = torch.empty((b, s, hq, d), dtype=dtype, device=device)
        return state
    if case["order"] == "bhsd":
        state["q"] = _normal((b, hq, s, d), dtype, gen).transpose(1, 2)
        state["k"] = _normal((b, hk, s, d), dtype, gen).transpose(1, 2)
    elif case["order"] == "qkv":
        fused = _normal((b, s, hq + 2 * hk, d), dtype, gen)
        state["q"], state["k"] = fused[:, :, :hq], fused[:, :, hq:hq + hk]
    else:
        state["q"], state["k"] = _normal((b, s, hq, d), dtype, gen), _normal((b, s, hk, d), dtype, gen)
    shift = torch.randint(0, 64, (b, 1), generator=gen, device=device)
    state["positions"] = case["start"] + shift + torch.arange(s, device=device)
    state["q_out"], state["k_out"] = torch.empty_like(state["q"]), torch.empty_like(state["k"])
    return state


def _prepare_sample(case, gen, dtype):
    rows, vocab, device = case["rows"], case["vocab"], gen.device

    def rand(*shape):
        return torch.rand(shape, generator=gen, device=device)

    logits = case["spread"] * torch.randn((rows, vocab), generator=gen, device=device)
    logits += 2.0 * case["spread"] * (rand(rows, vocab) < 4.0 / vocab)  # a few tokens that the model is sure of
    state = {"case": case, "logits": logits.to(dtype), "uniforms": rand(rows), "recent": None, "ignore": None}
    state["temperature"], state["top_k"] = case["temperature"], case["top_k"]
    state["top_p"], state["min_p"] = case["top_p"], case["min_p"]
    if case["per_row"]:  # requests with settings of their own: greedy ones, some with a top-k, some without a filter
        state["temperature"] = 0.5 + rand(rows)
        state["temperature"][rand(rows) < 0.1] = 0.0
        k = torch.randint(1, 400, (rows,), generator=gen, device=device)
        state["top_k"] = torch.where(rand(rows) < 0.3, k, 0)
        state["top_p"] = torch.where(rand(rows) < 0.8, 0.6 + 0.39 * rand(rows), 1.0)
        state["min_p"] = torch.where(rand(rows) < 0.3, 0.1 * rand(rows), 0.0)
    if case["recent"]:
        state["recent"] = torch.randint(-1, vocab, (rows, case["recent"]), generator=gen, device=device)
    if case["ignore"]:
        state["ignore"] = torch.randint(0, vocab, (case["ignore"],), generator=gen, device=device)
    state["tokens"] = torch.empty(rows, dtype=torch.int64, device=device)
    state["logprobs"] = torch.empty(rows, dtype=torch.float32, device=device)
    return state


PENALTY = 1.1
STREAMS = 3  # the ignore list holds for the first of each song's token streams


# --------------------------------------------------------------------------- one pass

def run(state):
    kind = state["case"]["kind"]
    if kind == "rope":
        return _run_rope(state)
    if kind == "append":
        return _run_append(state)
    return _run_sample(state)


def _run_rope(s):
    c = s["case"]
    if own:
        q, k = _ops().rope_qk_t(s["q"], s["k"], s["theta"], s["positions"], interleaved=c["interleaved"],
                                adjoint=c["adjoint"], magnitude=c["magnitude"], q_out=s["q_out"], k_out=s["k_out"])
        return {"q": q, "k": k}
    cos, sin = _turns(s["positions"], s["theta"], c["adjoint"], c["magnitude"])
    return {"q": _turn(s["q"], cos, sin, c["interleaved"]), "k": _turn(s["k"], cos, sin, c["interleaved"])}


def _run_append(s):
    c = s["case"]
    if own:
        q = _ops().rope_append_kv_t(s["q"], s["k"], s["v"], s["theta"], s["k_cache"], s["v_cache"], s["lengths"],
                                    counts=s["counts"], interleaved=c["interleaved"], q_out=s["q_out"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    at = torch.arange(c["seq"], device=s["q"].device)
    rows = s["lengths"][:, None] + at
    cos, sin = _turns(rows, s["theta"], False, 1.0)
    taken = (at < s["counts"][:, None]).nonzero(as_tuple=True)
    k = _turn(s["k"], cos, sin, c["interleaved"])
    s["k_cache"][taken[0], rows[taken]] = k[taken]
    s["v_cache"][taken[0], rows[taken]] = s["v"][taken]
    return {"q": _turn(s["q"], cos, sin, c["interleaved"]), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _turns(positions, theta, adjoint, magnitude):
    """Cosine and sine of every token's angles, in 64 bits up to the rounding to 32."""
    angle = positions[:, :, None, None].double() * theta
    cos, sin = (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()
    return cos, -sin if adjoint else sin


def _turn(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    y = x.float()
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)


def _run_sample(s):
    if own:
        tokens = _ops().sample_tokens_t(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"],
                                        top_p=s["top_p"], min_p=s["min_p"], recent=s["recent"], penalty=PENALTY,
                                        penalty_limit=s["case"]["vocab"] - 1, ignore=s["ignore"], streams=STREAMS,
                                        logprobs=s["logprobs"], out=s["tokens"])
        return {"tokens": tokens, "logprobs": s["logprobs"]}
    x = s["logits"].float()
    rows, vocab = x.shape
    if s["recent"] is not None:
        ids = torch.where(s["recent"] < vocab - 1, s["recent"], -1) + 1
        told = torch.zeros((rows, vocab + 1), dtype=torch.bool, device=x.device).scatter_(1, ids, True)[:, 1:]
        x = x / torch.where(told, PENALTY, 1.0)
    if s["ignore"] is not None:
        first = torch.arange(rows, device=x.device) % STREAMS == 0
        out = torch.zeros(vocab, dtype=torch.bool, device=x.device).index_fill_(0, s["ignore"], True)
        x = x.masked_fill(first[:, None] & out, -math.inf)

    def each(v):
        return v[:, None] if isinstance(v, torch.Tensor) else torch.full((rows, 1), v, device=x.device)

    temperature, top_k, top_p, min_p = (each(s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    value, index = x.sort(dim=1, descending=True, stable=True)
    rank = torch.arange(vocab, device=x.device)
    warm = torch.where(temperature > 0, temperature, 1.0).double()
    weight = ((value.double() - value[:, :1].double()) / warm).exp()
    weight *= (rank < torch.where(top_k > 0, top_k, vocab)) & ((temperature > 0) | (rank == 0))
    upto = weight.cumsum(1)
    before = torch.cat((torch.zeros_like(upto[:, :1]), upto[:, :-1]), 1)
    kept = ((before < top_p.double() * upto[:, -1:]) | (rank == 0)) & (weight >= min_p.double()) & (weight > 0)
    total = upto.gather(1, kept.sum(1, keepdim=True) - 1)
    place = (upto <= s["uniforms"][:, None].double() * total).sum(1, keepdim=True)
    place = torch.minimum(place, kept.sum(1, keepdim=True) - 1)
    return {"tokens": index.gather(1, place)[:, 0],
            "logprobs": (weight.gather(1, place) / total).log().float()[:, 0]}


# --------------------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "sample": _exact_sample}[case["kind"]](state)


def _host(t):
    return t.to("cpu", torch.float64).numpy()


def _exact_turn(x, positions, theta, interleaved, adjoint, magnitude):
    """Each pair as a complex number, times that of its angle."""
    rot = 2 * len(theta)
    spin = magnitude * np.exp((-1j if adjoint else 1j) * positions[:, :, None] * theta)[:, :, None, :]
    y = x.copy()
    if interleaved:
        z = (x[..., 0:rot:2] + 1j * x[..., 1:rot:2]) * spin
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    else:
        z = (x[..., :rot // 2] + 1j * x[..., rot // 2:rot]) * spin
        y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
    return y


def _exact_rope(s):
    c = s["case"]
    args = (_host(s["positions"]), _host(s["theta"]), c["interleaved"], c["adjoint"], c["magnitude"])
    return {n: torch.from_numpy(_exact_turn(_host(s[n]), *args)) for n in ("q", "k")}


def _exact_append(s):
    c = s["case"]
    lengths, counts = s["lengths"].cpu().numpy(), s["counts"].cpu().numpy()
    positions = (lengths[:, None] + np.arange(c["seq"])).astype(np.float64)
    args = (positions, _host(s["theta"]), c["interleaved"], False, 1.0)
    k, v = _exact_turn(_host(s["k"]), *args), _host(s["v"])
    k_cache, v_cache = np.zeros(s["k_cache"].shape), np.zeros(s["v_cache"].shape)
    for b, (start, n) in enumerate(zip(lengths, counts)):
        k_cache[b, start:start + n], v_cache[b, start:start + n] = k[b, :n], v[b, :n]
    return {"q": torch.from_numpy(_exact_turn(_host(s["q"]), *args)), "k_cache": torch.from_numpy(k_cache),
            "v_cache": torch.from_numpy(v_cache)}


def _exact_sample(s):
    """Row by row: order, the three filters one after the other, the inverse of the distribution function."""
    rows, vocab = s["logits"].shape
    if rows * vocab > 1 << 25:
        return None
    logits = s["logits"].float().cpu().numpy()

    def each(v):
        return v.cpu().numpy().tolist() if isinstance(v, torch.Tensor) else [float(np.float32(v))] * rows

    settings = zip(*(each(s[n]) for n in ("temperature", "top_k", "top_p", "min_p", "uniforms")))
    tokens, logprobs = np.zeros(rows, np.int64), np.zeros(rows)
    for r, (temperature, top_k, top_p, min_p, uniform) in enumerate(settings):
        x = logits[r].copy()
        if s["recent"] is not None:
            told = np.unique(s["recent"][r].cpu().numpy())
            told = told[(told >= 0) & (told < vocab - 1)]
            x[told] = x[told] / np.float32(PENALTY)
        if s["ignore"] is not None and r % STREAMS == 0:
            x[s["ignore"].cpu().numpy()] = -np.inf
        order = np.argsort(-x, kind="stable")
        if temperature == 0:
            order = order[:1]
        if top_k > 0:
            order = order[:int(top_k)]
        p = np.exp((x[order].astype(np.float64) - float(x[order[0]])) / (temperature or 1.0))
        keep = len(p)
        if top_p < 1:
            keep = max(1, int(np.sum(np.cumsum(p) - p < top_p * p.sum())))
        keep = min(keep, int(np.sum(p >= min_p)))
        p = p[:keep] / p[:keep].sum()
        at = min(int(np.searchsorted(np.cumsum(p), uniform, side="right")), keep - 1)
        tokens[r], logprobs[r] = order[at], math.log(p[at])
    return {"tokens": torch.from_numpy(tokens), "logprobs": torch.from_numpy(logprobs)}
