"""Sampling against the 64-bit definition: equal tokens, at the sizes, ties, masks and settings where it can go
wrong; and the distribution that a grid of uniform numbers draws."""
from __future__ import annotations

import math
import subprocess
import sys

import numpy as np
import pytest
import torch

from conftest import ROOT
from token_step_reference import DTYPES, logprob_tolerance, penalised, sample_row

pytestmark = pytest.mark.gpu
VOCAB = 16385  # LeLM codebook 16384 + EOS


def run(ops, logits, u, dev, **kw):
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    logprobs = torch.empty(logits.shape[0], device=dev)
    tokens = ops.sample_tokens_t(logits, u, logprobs=logprobs, status=status, **kw)
    return tokens.cpu().numpy(), logprobs.cpu().numpy().astype(np.float64), status.item()


def check(ops, dev, logits, u, expect_status=0, **kw):
    """Tokens equal to the definition's and logprobs within the rounding of the weights; status as expected, with
    SAMPLE_EMPTY where the definition finds a row without a token."""
    tokens, logprobs, status = run(ops, logits, u, dev, **kw)
    rows, vocab = logits.shape
    x = penalised(logits, None if kw.get("recent") is None else kw["recent"].cpu().numpy(), kw.get("penalty", 1.0),
                  kw.get("penalty_limit", 0), None if kw.get("ignore") is None else kw["ignore"].cpu().numpy(),
                  kw.get("streams", 0))

    def each(name, off):
        v = kw.get(name, off)
        return v.cpu().tolist() if isinstance(v, torch.Tensor) else [float(np.float32(v))] * rows

    settings = zip(each("temperature", 1.0), [int(k) for k in each("top_k", 0)], each("top_p", 1.0),
                   each("min_p", 0.0), u.cpu().tolist())
    for r, (temperature, top_k, top_p, min_p, uniform) in enumerate(settings):
        want = sample_row(x[r], uniform, temperature, top_k, top_p, min_p)
        if want is None:
            expect_status |= ops.SAMPLE_EMPTY
            assert tokens[r] == 0 and logprobs[r] == -np.inf
            continue
        token, logprob, weight, total, near = want
        assert tokens[r] == token, f"row {r}: {tokens[r]}, not {token} ({near:.3g} from a border)"
        tol = logprob_tolerance(logprob, weight, total, vocab)
        assert abs(logprobs[r] - logprob) <= tol, f"row {r}: logprob {logprobs[r]} not {logprob} +- {tol}"
    assert status == expect_status
    return tokens


def uniforms(gen, rows):
    return torch.rand(rows, generator=gen, device=gen.device)


FILTERS = {
    "none": {}, "k1": {"top_k": 1}, "k50": {"top_k": 50}, "k1500": {"top_k": 1500}, "k over": {"top_k": 10 ** 9},
    "p0": {"top_p": 0.0}, "p50": {"top_p": 0.5}, "p999": {"top_p": 0.999}, "m0.1": {"min_p": 0.1}, "m1": {"min_p": 1.0},
    "k+p": {"top_k": 200, "top_p": 0.9}, "all": {"top_k": 300, "top_p": 0.95, "min_p": 0.01, "temperature": 0.7},
    "hot": {"temperature": 20.0, "top_p": 0.9}, "cold": {"temperature": 0.01}, "zero": {"temperature": 0.0},
    "k+m": {"top_k": 40, "min_p": 0.05},
}


@pytest.mark.parametrize("name", FILTERS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, VOCAB, 50257])
def test_sample_matches_definition(ops, dev, dtype, vocab, name):
    gen = torch.Generator(device=dev).manual_seed(vocab + len(name))
    logits = (3.0 * torch.randn((5, vocab), generator=gen, device=dev)).to(DTYPES[dtype])
    check(ops, dev, logits, uniforms(gen, 5), **FILTERS[name])


@pytest.mark.parametrize("vocab,rows", [(131072, 1), (131071, 3), (100003, 9), (65536, 2)])
@pytest.mark.parametrize("name", ["none", "k50", "k1500", "p999", "all", "hot", "m0.1"])
def test_sample_large_vocabularies(ops, dev, vocab, rows, name):
    gen = torch.Generator(device=dev).manual_seed(vocab + rows)
    logits = (2.0 * torch.randn((rows, vocab), generator=gen, device=dev)).bfloat16()
    check(ops, dev, logits, uniforms(gen, rows), **FILTERS[name])


@pytest.mark.parametrize("rows", [1, 2, 7, 149, 600])
def test_sample_row_counts(ops, dev, rows):
    gen = torch.Generator(device=dev).manual_seed(rows)
    logits = 2.5 * torch.randn((rows, 2000), generator=gen, device=dev)
    check(ops, dev, logits, uniforms(gen, rows), top_k=100, top_p=0.9)
    check(ops, dev, logits, uniforms(gen, rows), top_p=0.9)


def test_sample_settings_of_each_row(ops, dev):
    gen = torch.Generator(device=dev).manual_seed(1)
    rows = 64
    logits = (3 * torch.randn((rows, VOCAB), generator=gen, device=dev)).half()
    temperature = 0.3 + 1.5 * uniforms(gen, rows)
    temperature[::7] = 0.0
    top_k = torch.randint(0, 3000, (rows,), generator=gen, device=dev)
    top_k[::3] = 0
    top_p = uniforms(gen, rows)
    top_p[::4] = 1.0
    min_p = 0.2 * uniforms(gen, rows)
    min_p[::2] = 0.0
    check(ops, dev, logits, uniforms(gen, rows), temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["none", "k50", "k1500", "p50", "all"])
def test_sample_ties(ops, dev, dtype, name):
    """Equal logits are taken by index, inside and at the border of every filter."""
    gen = torch.Generator(device=dev).manual_seed(2)
    rows = 12
    few = torch.randint(0, 9, (rows, VOCAB), generator=gen, device=dev).to(DTYPES[dtype])
    few[0] = 1.5                                  # all equal
    few[1] = 0.0
    few[1, ::2] = -0.0                            # zeros of both signs are equal
    few[2] = torch.where(torch.arange(VOCAB, device=dev) % 1000 == 7, 5.0, 0.0).to(few.dtype)
    few[3, 100:] = -math.inf
    check(ops, dev, few, uniforms(gen, rows), **FILTERS[name])


@pytest.mark.parametrize("name", ["none", "k50", "k1500", "p50", "p999", "all", "m0.1"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_masked_rows(ops, dev, dtype, name):
    """-inf, the type's lowest value, +inf, one token left, none left, a wide range of magnitudes."""
    gen = torch.Generator(device=dev).manual_seed(3)
    t, vocab = DTYPES[dtype], 5000
    x = (3 * torch.randn((9, vocab), generator=gen, device=dev)).to(t)
    x[0, 1:] = -math.inf
    x[1, :-1] = torch.finfo(t).min
    x[2, ::3] = -math.inf
    x[3, torch.arange(vocab, device=dev) % 50 != 3] = torch.finfo(t).min
    x[4] = torch.finfo(t).min
    x[5, [10, 3000, 77]] = math.inf
    x[6] = -math.inf
    x[7] = (x[7].float() * 1e4).clamp(-6e4, 6e4).to(t)
    x[8] = (x[8].float() * 1e-6).to(t)
    check(ops, dev, x, uniforms(gen, 9), expect_status=ops.SAMPLE_EMPTY, **FILTERS[name])


def test_sample_clusters_of_close_logits(ops, dev):
    """Thousands of different logits within few units of the last place, beside wide ones: no bin splits them at once."""
    gen = torch.Generator(device=dev).manual_seed(4)
    vocab = 20000
    base = torch.full((6, vocab), 7.0, device=dev)
    base += torch.randint(0, 4000, (6, vocab), generator=gen, device=dev) * 2.0 ** -21
    base[1, ::2] -= 25.0
    base[2] *= 1e-30
    base[3, 0] = 30.0
    base[4, 5:9000] = -3e38
    base[5, 7] = 7.5
    for name in ("none", "k1500", "p50", "k+p", "m0.1"):
        check(ops, dev, base, uniforms(gen, 6), **FILTERS[name])
    check(ops, dev, base, uniforms(gen, 6), top_k=9999, top_p=0.7)
    check(ops, dev, base, uniforms(gen, 6), temperature=1e-6)
    check(ops, dev, base, uniforms(gen, 6), temperature=1e6, top_p=0.3)


# Rows x vocabulary by how a row is worked on: one CTA that holds it (few rows, many, a long row); one that reads it
# again; a cluster of eight that holds its shares (few rows, many), of four; one of four that reads them again, and of
# two; one list.
SHARES = [(7, 16385), (200, 16385), (6, 32700), (300, 20011), (2, 131072), (30, 131072), (5, 50257), (40, 131071),
          (100, 50257), (9, 512)]


@pytest.mark.parametrize("rows,vocab", SHARES)
@pytest.mark.parametrize("name", ["none", "k50", "k1500", "p999", "all", "m0.1", "zero"])
def test_sample_hard_rows_whatever_the_split(ops, dev, rows, vocab, name):
    """Ties, masks, infinities and edited ids in every split of the work; the edited ids lie at the shares' ends too."""
    gen = torch.Generator(device=dev).manual_seed(vocab + rows)
    t = list(DTYPES.values())[rows % 3]
    x = (2 * torch.randn((rows, vocab + 3), generator=gen, device=dev)).to(t)[:, 1:vocab + 1]
    x[0] = torch.randint(0, 5, (vocab,), generator=gen, device=dev).to(t)        # thousands of equal logits
    x[1, ::2] = -math.inf
    if rows > 2:
        x[2] = 0.25
        x[3, 5:vocab - 2] = torch.finfo(t).min
        x[4, torch.randint(0, vocab, (3,), generator=gen, device=dev)] = math.inf
    if rows > 6:
        x[5] = (x[5].float() * 1e-4 + 9).to(t)
        x[6, :-1] = -math.inf
    edges = torch.tensor([0, 1, vocab // 2 - 1, vocab // 2, vocab - 1, vocab - 2, -1, vocab + 5], device=dev)
    recent = torch.cat((edges.expand(rows, -1), torch.randint(-1, vocab, (rows, 600), generator=gen, device=dev)), 1)
    top = x.float().topk(3, dim=1).indices
    recent = torch.cat((recent, top), 1).contiguous()
    ignore = torch.cat((edges, top[0], torch.randint(0, vocab, (700,), generator=gen, device=dev)))
    u = uniforms(gen, rows)
    check(ops, dev, x, u, **FILTERS[name])
    check(ops, dev, x, u, recent=recent, penalty=1.2, penalty_limit=vocab - 1, ignore=ignore, streams=2, **FILTERS[name])


@pytest.mark.parametrize("rows,vocab", SHARES)
def test_sample_nan_whatever_the_split(ops, dev, rows, vocab):
    gen = torch.Generator(device=dev).manual_seed(rows)
    x = torch.randn((rows, vocab), generator=gen, device=dev)
    u = uniforms(gen, rows)
    for place in (0, vocab // 3, vocab - 1):
        y = x.clone()
        y[rows - 1, place] = math.nan
        check(ops, dev, y, u, expect_status=ops.SAMPLE_NAN, top_p=0.9)
        listed = torch.tensor([place], device=dev)
        check(ops, dev, y, u, ignore=listed, streams=1, top_k=30)  # an ignored NaN is no NaN
        y[rows - 1] = math.nan
        check(ops, dev, y, u, expect_status=ops.SAMPLE_NAN | ops.SAMPLE_EMPTY, top_k=3)


def test_sample_nan(ops, dev):
    x = torch.zeros((3, 100), device=dev)
    x[1, 42] = math.nan
    x[2, 5] = math.nan
    u = torch.full((3,), 0.425, device=dev)
    tokens, logprobs, status = run(ops, x, u, dev, ignore=torch.tensor([5], device=dev), streams=2)
    assert status == ops.SAMPLE_NAN                 # row 1's; row 2's NaN is on its ignore list
    assert tokens.tolist() == [43, 43, 43]          # 99 tokens each; row 0 without 5, row 1 without 42, row 2 without 5
    assert np.allclose(logprobs, math.log(1 / 99), atol=1e-6)
    x = torch.full((1, 50), math.nan, device=dev)
    assert run(ops, x, u[:1], dev)[2] == ops.SAMPLE_NAN | ops.SAMPLE_EMPTY


def test_sample_values_out_of_range(ops, dev):
    """Counted as the header says, and flagged."""
    rows, vocab = 10, 300
    gen = torch.Generator(device=dev).manual_seed(5)
    x = 2 * torch.randn((rows, vocab), generator=gen, device=dev)
    u = torch.full((rows,), 0.5, device=dev)
    one = {"temperature": [1.0] * rows, "top_k": [0] * rows, "top_p": [1.0] * rows, "min_p": [0.0] * rows}
    given = {n: list(v) for n, v in one.items()}
    taken = {n: list(v) for n, v in one.items()}
    for r, (n, bad, good) in enumerate((("temperature", -1.0, 0.0), ("temperature", math.nan, 0.0),
                                        ("temperature", math.inf, 0.0), ("top_k", -3, 0), ("top_p", math.nan, 1.0),
                                        ("top_p", -0.5, 0.0), ("top_p", 2.0, 1.0), ("min_p", math.nan, 0.0),
                                        ("min_p", 3.0, 1.0), ("min_p", -1.0, 0.0))):
        given[n][r], taken[n][r] = bad, good

    def tensors(d):
        return {n: torch.tensor(v, device=dev, dtype=torch.int64 if n == "top_k" else torch.float32)
                for n, v in d.items()}

    tokens, logprobs, status = run(ops, x, u, dev, **tensors(given))
    want, want_lp, clean = run(ops, x, u, dev, **tensors(taken))
    assert status == ops.SAMPLE_PARAM and clean == 0
    assert np.array_equal(tokens, want) and np.array_equal(logprobs, want_lp)
    for r in range(rows):
        alone = {n: v[r:r + 1] for n, v in tensors(given).items()}
        assert run(ops, x[r:r + 1], u[r:r + 1], dev, **alone)[2] == ops.SAMPLE_PARAM, r
    edge = torch.tensor([0.0, 1.0, 7.0, -1.0, math.nan], device=dev)
    tokens, _, status = run(ops, x[:1].expand(5, vocab).contiguous(), edge, dev, top_k=10)
    order = torch.sort(x[0], descending=True).indices.tolist()
    assert status == ops.SAMPLE_PARAM and tokens.tolist() == [order[0], order[9], order[9], order[0], order[0]]


def test_sample_penalty_and_ignore_list(ops, dev):
    gen = torch.Generator(device=dev).manual_seed(6)
    rows = 12
    x = 3 * torch.randn((rows, VOCAB), generator=gen, device=dev)
    recent = torch.randint(-1, VOCAB, (rows, 700), generator=gen, device=dev)
    recent[:, ::5] = recent[:, 1:2]  # repeats count once
    top = x.topk(8, dim=1).indices
    recent[:, 2:10] = top
    recent[0, 3] = 2 ** 40
    ignore = torch.cat((top[0, :3], top[3, :2], torch.tensor([-5, VOCAB, 2 ** 33], device=dev)))
    u = uniforms(gen, rows)
    for streams in (0, 1, 3):
        check(ops, dev, x, u, recent=recent, penalty=1.3, penalty_limit=VOCAB - 1, ignore=ignore, streams=streams,
              top_k=20, top_p=0.9)
        check(ops, dev, x, u, recent=recent, penalty=0.7, ignore=ignore, streams=streams, top_p=0.95)
    everything = torch.arange(VOCAB, device=dev)
    tokens, _, status = run(ops, x, u, dev, ignore=everything, streams=rows)
    assert tokens[0] == 0 and status == ops.SAMPLE_EMPTY


def test_sample_at_temperature_zero_is_the_greedy_choice(ops, dev):
    gen = torch.Generator(device=dev).manual_seed(7)
    x = torch.randint(0, 40, (9, VOCAB), generator=gen, device=dev).float()
    recent = torch.randint(-1, VOCAB, (9, 50), generator=gen, device=dev)
    ignore = torch.randint(0, VOCAB, (16,), generator=gen, device=dev)
    kw = {"recent": recent, "penalty": 1.1, "penalty_limit": VOCAB - 1, "ignore": ignore}
    want = ops.greedy_tokens_t(x, **kw)
    got = ops.sample_tokens_t(x, uniforms(gen, 9), temperature=0.0, **kw)
    assert torch.equal(got, want)


def test_sample_strided_rows_and_neighbours(ops, dev):
    gen = torch.Generator(device=dev).manual_seed(8)
    for t in DTYPES.values():
        big = (3 * torch.randn((7, 3007), generator=gen, device=dev)).to(t)
        for lo, hi in ((0, 3000), (1, 2998), (3, 2500)):
            check(ops, dev, big[:, lo:hi], uniforms(gen, 7), top_p=0.9)
            check(ops, dev, big[:, lo:hi], uniforms(gen, 7), top_k=64)
    out = torch.full((9,), -7, dtype=torch.int64, device=dev)
    lp = torch.full((9,), 5.0, device=dev)
    ops.sample_tokens_t(big, uniforms(gen, 7), out=out[1:8], logprobs=lp[1:8])
    assert out[0] == out[8] == -7 and lp[0] == lp[8] == 5.0


@pytest.mark.parametrize("kw", [{}, {"top_k": 12}, {"top_p": 0.8}, {"min_p": 0.05}])
def test_sample_draws_the_distribution(ops, dev, kw):
    """A grid of n uniform numbers gives each kept token n p rounded down or up, and no other."""
    gen = torch.Generator(device=dev).manual_seed(9)
    n, vocab = 20000, 40
    x = 1.5 * torch.randn((1, vocab), generator=gen, device=dev)
    u = (torch.arange(n, device=dev) + 0.5) / n
    tokens = ops.sample_tokens_t(x.expand(n, vocab).contiguous(), u, **kw).cpu().numpy()
    drawn = np.bincount(tokens, minlength=vocab)
    row = x[0].cpu().numpy()
    order = np.argsort(-row, kind="stable")
    p = np.exp(row[order].astype(np.float64) - row.max())
    keep = vocab
    if "top_k" in kw:
        keep = 12
    if "top_p" in kw:
        keep = int(np.sum(np.cumsum(p) - p < np.float32(0.8) * p.sum()))
    if "min_p" in kw:
        keep = int(np.sum(p >= np.float32(0.05)))
    want = np.zeros(vocab)
    want[order[:keep]] = p[:keep] / p[:keep].sum()
    assert np.all(np.abs(drawn - n * want) <= 1.0 + 1e-3)  # the grid is F32: 1e-3 of a step off
    assert np.all(drawn[order[keep:]] == 0)


def test_sample_captured_and_replayed_beside_another_graph(ops, dev):
    gen = torch.Generator(device=dev).manual_seed(10)
    rows = 4
    cases = []
    for vocab, kw in ((VOCAB, {"top_k": 50}), (131072, {"top_p": 0.9}), (VOCAB, {"top_p": 0.95, "min_p": 0.01})):
        x, u = torch.empty((rows, vocab), device=dev), torch.empty(rows, device=dev)
        out = torch.empty(rows, dtype=torch.int64, device=dev)
        x.normal_(generator=gen)
        u.uniform_(generator=gen)
        ops.sample_tokens_t(x, u, out=out, **kw)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.sample_tokens_t(x, u, out=out, **kw)
        cases.append((graph, x, u, out, kw))
    for _ in range(3):
        for _, x, u, _, _ in cases:
            x.normal_(generator=gen)
            u.uniform_(generator=gen)
        for graph, *_ in cases:
            graph.replay()
        torch.cuda.synchronize()
        for _, x, u, out, kw in cases:
            assert torch.equal(out, ops.sample_tokens_t(x, u, **kw))


def test_sample_first_call_of_a_process_under_capture(dev):
    """Kernels are loaded and opt in to their shared memory inside a capture, without a call before it."""
    code = (
        "import sys; sys.path.insert(0, %r); import torch, __graft_entry__ as e; ops = e.load_package().ops\n"
        "x, u = torch.randn(3, 16385, device='cuda'), torch.rand(3, device='cuda')\n"
        "q = torch.randn(2, 700, 12, 128, device='cuda', dtype=torch.float16)\n"
        "out, turned = torch.zeros(3, dtype=torch.int64, device='cuda'), torch.empty_like(q)\n"
        "theta = ops.rope_theta(128, device='cuda')\n"
        "g = torch.cuda.CUDAGraph()\n"
        "with torch.cuda.graph(g):\n"
        "    ops.sample_tokens_t(x, u, top_p=0.9, out=out); ops.rope_qk_t(q, None, theta, q_out=turned)\n"
        "g.replay(); torch.cuda.synchronize()\n"
        "assert torch.equal(out, ops.sample_tokens_t(x, u, top_p=0.9))\n"
        "assert torch.equal(turned, ops.rope_qk_t(q, None, theta)[0]); print('captured')\n" % str(ROOT))
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_sample_is_the_same_every_time_and_on_other_streams(ops, dev):
    gen = torch.Generator(device=dev).manual_seed(11)
    x = torch.randn((300, VOCAB), generator=gen, device=dev)
    u = uniforms(gen, 300)
    lp = torch.empty(300, device=dev)
    want = ops.sample_tokens_t(x, u, top_p=0.97, logprobs=lp)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(3)]
    results = []
    for stream in streams:
        with torch.cuda.stream(stream):
            for _ in range(3):
                again = torch.empty(300, device=dev)
                results.append((ops.sample_tokens_t(x, u, top_p=0.97, logprobs=again), again))
    torch.cuda.synchronize()
    for tokens, again in results:
        assert torch.equal(tokens, want) and torch.equal(again, lp)


def test_sample_on_a_device_that_is_not_current(ops, dev):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    other = torch.device("cuda:1")
    gen = torch.Generator(device=dev).manual_seed(12)
    x, u = torch.randn((3, 1000), generator=gen, device=dev), uniforms(gen, 3)
    got = ops.sample_tokens_t(x.to(other), u.to(other), top_k=20)
    assert got.device == other and torch.equal(got.cpu(), ops.sample_tokens_t(x, u, top_k=20).cpu())
    with pytest.raises(ValueError, match="one CUDA device"):
        ops.sample_tokens_t(x, u.to(other))


def test_sample_no_rows(ops, dev):
    assert ops.sample_tokens_t(torch.empty((0, 10), device=dev), torch.empty(0, device=dev)).shape == (0,)


# Vocabularies that one CTA reads: held, read again with many rows of two CTAs an SM, in one or several rounds of loads.
@pytest.mark.parametrize("rows,vocab", [(160, 16384), (160, 2048), (320, 20480)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sample_extremes_in_every_warps_share(ops, dev, dtype, rows, vocab):
    """Rows without edited ids: the largest and the smallest logit, and a NaN, in the share of each warp in turn
    (a thread reads 16 bytes, a warp 512, sixteen warps one after the other), whichever warp comes first."""
    gen = torch.Generator(device=dev).manual_seed(vocab)
    t = DTYPES[dtype]
    of_warp = 512 // torch.empty(0, dtype=t).element_size()
    x = torch.randn((rows, vocab), generator=gen, device=dev).to(t)
    r = torch.arange(rows, device=dev)
    inside = torch.randint(0, of_warp, (2, rows), generator=gen, device=dev)
    most = (r % 16 * of_warp + inside[0]) % vocab
    least = ((r // 16 + r + 5) % 16 * of_warp + inside[1]) % vocab
    x[r, least] = -9.0
    x[r, most] = 9.0
    for name in ("none", "k50", "p50", "m0.1", "hot", "zero"):
        check(ops, dev, x, uniforms(gen, rows), **FILTERS[name])
    # a NaN in one row: the flag, and the token of the others
    for row in range(0, 32, 3):
        y = x.clone()
        y[row, least[row]] = math.nan
        status = torch.zeros(1, dtype=torch.int32, device=dev)
        tokens = ops.sample_tokens_t(y, uniforms(gen, rows), temperature=0.0, status=status)
        assert status.item() == ops.SAMPLE_NAN and torch.equal(tokens, most)


@pytest.mark.parametrize("rows,vocab", [(18, 32768), (37, 32800), (18, 131072), (60, 50257)])
def test_sample_split_rows_behind_and_beside_other_work(ops, dev, rows, vocab):
    """CTAs of a cluster that start late and read little: behind products that fill the SMs, on several streams at
    once, with nothing to edit and with everything masked but a share's end."""
    gen = torch.Generator(device=dev).manual_seed(rows + vocab)
    x = (2 * torch.randn((rows, vocab), generator=gen, device=dev)).bfloat16()
    x[0, :-1] = -math.inf
    x[1, 1:] = -math.inf
    u = uniforms(gen, rows)
    want = torch.from_numpy(check(ops, dev, x, u, top_p=0.9))
    a = torch.randn((2048, 2048), generator=gen, device=dev)
    streams = [torch.cuda.Stream(device=dev) for _ in range(3)]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream(dev))
    results = []
    for _ in range(20):
        for stream in streams:
            with torch.cuda.stream(stream):
                a @ a
                results += [ops.sample_tokens_t(x, u, top_p=0.9) for _ in range(2)]
    torch.cuda.synchronize()
    for tokens in results:
        assert torch.equal(tokens.cpu(), want)


@pytest.mark.parametrize("rows,vocab", [(7, 16385), (200, 5000), (300, 20011), (7, 131072), (9, 512)])
@pytest.mark.parametrize("temperature", [1e-30, 1e-36, 1e-37, 3e-38, 1e-38, 1e-41, 1e-45])
def test_sample_tiny_temperatures(ops, dev, rows, vocab, temperature):
    """Logits so near the top that a temperature below F32's normal range still tells them apart, and others that
    lie thousands of temperatures below it: those have no weight, whatever slice they fall into."""
    rng = np.random.default_rng(rows + vocab)
    x = np.zeros((rows, vocab), np.float64)
    for r in range(rows):
        near = rng.random(vocab)
        x[r] = (-2.3e-35 * near, -300 * temperature * near, 3e-36 * near, -2.0 ** -149 * rng.integers(0, 9000, vocab),
                np.floor(4 * near), np.where(near < 0.5, -40 * temperature * near, -3e38),
                np.where(near < 0.01, -3 * temperature * rng.random(vocab), -2.4e-35 * near))[r % 7]
    x[5::7, ::3] = -np.inf
    logits = torch.from_numpy(x.astype(np.float32)).to(dev)
    gen = torch.Generator(device=dev).manual_seed(vocab)
    for name in ("none", "k50", "k1500", "p50", "p999", "m0.1", "k+p"):
        check(ops, dev, logits, uniforms(gen, rows), temperature=temperature, **FILTERS[name])


def plain_choice(x, u, temperature, top_k, top_p, min_p):
    """The definition with plain F64 sums, nothing rounded to a unit: (token, log of its share, bound on the error of
    that log), or None where a border lies so near that the documented unit may decide it."""
    unit = 2.0 * 2.0 ** -44  # a weight's rounding to 2^-44 and the error of the exponential before it
    order = np.argsort(-x, kind="stable")
    if top_k:
        order = order[:top_k]
    v = x[order].astype(np.float64)
    w = np.exp((v - v[0]) / temperature)
    upto = np.cumsum(w)
    slack = len(w) * (unit + 2.0 ** -53 * upto[-1])  # of a sum: the units', and this one's own roundings
    keep = len(w)
    if top_p < 1:
        target = top_p * upto[-1]
        if np.min(np.abs(upto - target)) <= 2 * slack:
            return None
        keep = max(1, int(np.sum(upto - w < target)))
    if min_p > 0:
        if np.min(np.abs(w - min_p)) <= unit:
            return None
        keep = min(keep, int(np.sum(w >= min_p)))
    target = u * upto[keep - 1]
    if np.min(np.abs(upto - target)) <= 2 * slack:
        return None
    at = min(int(np.searchsorted(upto, target, side="right")), keep - 1)
    logprob = math.log(w[at] / upto[keep - 1])
    return int(order[at]), logprob, 2.0 ** -24 * abs(logprob) + 2 * unit / w[at] + 2 * slack / upto[keep - 1]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["none", "k50", "k1500", "p50", "p999", "m0.1", "k+p", "all", "hot"])
def test_sample_matches_plain_sums(ops, dev, dtype, name):
    """Where no border lies within the weights' unit, the unit does not show."""
    gen = torch.Generator(device=dev).manual_seed(21)
    rows, vocab = 96, VOCAB
    logits = (torch.linspace(0.3, 4.0, rows, device=dev)[:, None]
              * torch.randn((rows, vocab), generator=gen, device=dev)).to(DTYPES[dtype])
    u = uniforms(gen, rows)
    kw = FILTERS[name]
    tokens, logprobs, status = run(ops, logits, u, dev, **kw)
    x, near = logits.float().cpu().numpy(), 0
    for r in range(rows):
        want = plain_choice(x[r], float(u[r]), float(np.float32(kw.get("temperature", 1.0))), kw.get("top_k", 0),
                            float(np.float32(kw.get("top_p", 1.0))), float(np.float32(kw.get("min_p", 0.0))))
        if want is None:
            near += 1
            continue
        token, logprob, tol = want
        assert tokens[r] == token and abs(logprobs[r] - logprob) <= tol, r
    assert status == 0 and near <= rows // 8
