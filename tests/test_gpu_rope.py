"""Rotary positions and the KV append against the 64-bit definition: layouts, types, partial heads, odd sizes,
strides, far positions, the adjoint, ragged chunks, graphs and streams."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from token_step_reference import DTYPES, assert_rope, host, rope

pytestmark = pytest.mark.gpu


def make(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device=gen.device).to(dtype)


def check_qk(ops, q, k, theta, positions, dtype, **kw):
    """One call with fresh outputs against the definition; returns the outputs."""
    qo, ko = ops.rope_qk_t(q, k, theta, positions, **kw)
    b, s = q.shape[:2]
    pos = (torch.arange(s) + kw.get("start", 0)) if positions is None else positions.cpu()
    pos = np.broadcast_to(pos.numpy(), (b, s))
    th = theta.cpu().numpy()
    far = float(np.abs(pos).max() * th.max()) if s and b else 0.0
    ref = {n: kw[n] for n in ("interleaved", "adjoint", "magnitude") if n in kw}
    for name, x, y in (("q", q, qo), ("k", k, ko)):
        if x is None:
            continue
        want, size = rope(host(x), pos, th, **ref)
        assert_rope(y, want, size, dtype, far, name)
    return qo, ko


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,s,hq,hk,d,rot", [
    (1, 1, 1, 1, 2, 2), (2, 1, 12, 12, 128, 128), (1, 7, 3, 1, 64, 32), (2, 33, 20, 20, 110, 110), (3, 5, 4, 2, 96, 24),
    (1, 130, 8, 2, 80, 80), (2, 9, 5, 1, 256, 64), (1, 3, 2, 2, 18, 6), (1, 2, 1, 1, 1030, 1024), (1, 17, 33, 3, 48, 16),
    (1, 4, 2, 1, 72, 40), (2, 300, 2, 1, 128, 96),
])
def test_rope_matches_definition(ops, dev, dtype, interleaved, b, s, hq, hk, d, rot):
    gen = torch.Generator(device=dev).manual_seed(b * 1000 + s * 10 + d)
    t = DTYPES[dtype]
    q, k = make(gen, (b, s, hq, d), t), make(gen, (b, s, hk, d), t)
    positions = torch.randint(0, 5000, (b, s), generator=gen, device=dev)
    theta = ops.rope_theta(rot, device=dev)
    check_qk(ops, q, k, theta, positions, t, interleaved=interleaved)
    check_qk(ops, q, k, theta, positions, t, interleaved=interleaved, adjoint=True, magnitude=1.25)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("order", ["qkv", "bhsd", "offset", "odd token stride", "broadcast"])
def test_rope_layouts(ops, dev, dtype, order):
    gen = torch.Generator(device=dev).manual_seed(5)
    t, b, s, hq, hk, d = DTYPES[dtype], 2, 37, 6, 2, 64
    theta = ops.rope_theta(d, device=dev)
    if order == "qkv":
        fused = make(gen, (b, s, hq + 2 * hk, d), t)
        q, k = fused[:, :, :hq], fused[:, :, hq:hq + hk]
    elif order == "bhsd":
        q, k = make(gen, (b, hq, s, d), t).transpose(1, 2), make(gen, (b, hk, s, d), t).transpose(1, 2)
    elif order == "offset":  # one element off any wider alignment
        q = make(gen, (b * s * hq * d + 1,), t)[1:].view(b, s, hq, d)
        k = make(gen, (b * s * hk * d + 3,), t)[3:].view(b, s, hk, d)
    elif order == "odd token stride":
        q = make(gen, (b, s, hq * d + 5), t)[:, :, 1:hq * d + 1].unflatten(2, (hq, d))
        k = make(gen, (b, s, hk * d + 2), t)[:, :, 2:].unflatten(2, (hk, d))
    else:  # one head's values for all heads, one row of positions for the whole batch
        q = make(gen, (b, s, 1, d), t).expand(b, s, hq, d)
        k = make(gen, (1, s, hk, d), t).expand(b, s, hk, d)
    positions = torch.arange(s, device=dev) * 3
    check_qk(ops, q, k, theta, positions, t)
    check_qk(ops, q, k, theta, None, t, start=11, interleaved=True)
    check_qk(ops, q, None, theta, positions.expand(b, s), t)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rot", [64, 20])
def test_rope_in_place_and_into_a_larger_buffer(ops, dev, dtype, rot):
    gen = torch.Generator(device=dev).manual_seed(6)
    t, b, s, h, d = DTYPES[dtype], 2, 19, 3, 64
    q, k = make(gen, (b, s, h, d), t), make(gen, (b, s, 1, d), t)
    theta = ops.rope_theta(rot, device=dev)
    want_q, want_k = ops.rope_qk_t(q, k, theta, start=4)
    room = make(gen, (b, s + 2, h + 1, d + 3), t)
    before = room.clone()
    view = room[:, 1:s + 1, :h, 2:d + 2]
    ops.rope_qk_t(q, None, theta, start=4, q_out=view)
    assert torch.equal(view, want_q)
    view.copy_(before[:, 1:s + 1, :h, 2:d + 2])
    assert torch.equal(room, before)  # nothing beside the view was written
    q2, k2 = q.clone(), k.clone()
    ops.rope_qk_t(q2, k2, theta, start=4, q_out=q2, k_out=k2)
    assert torch.equal(q2, want_q) and torch.equal(k2, want_k)


@pytest.mark.parametrize("start", [0, 12345, 10 ** 6, 2 ** 30, -7])
def test_rope_far_positions(ops, dev, start):
    gen = torch.Generator(device=dev).manual_seed(7)
    q = make(gen, (1, 50, 2, 128), torch.float32)
    theta = ops.rope_theta(128, device=dev)
    check_qk(ops, q, None, theta, None, torch.float32, start=start)
    check_qk(ops, q, None, ops.rope_theta(128, scaling="by_parts", factor=8.0, device=dev), None, torch.float32,
             start=start)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_adjoint_is_the_gradient(ops, dev, interleaved):
    """Of the loss sum(g * y): against autograd of the formula in 64 bits, and against differences of the forward
    kernel (the map is linear, so a difference over a unit step is exact but for the two F32 roundings)."""
    gen = torch.Generator(device=dev).manual_seed(8)
    b, s, h, d, rot, m = 2, 5, 3, 32, 24, 1.2
    x, g = make(gen, (b, s, h, d), torch.float32), make(gen, (b, s, h, d), torch.float32)
    theta = ops.rope_theta(rot, device=dev)
    grad, _ = ops.rope_qk_t(g, None, theta, adjoint=True, interleaved=interleaved, magnitude=m)

    leaf = x.double().requires_grad_()
    phi = torch.arange(s, device=dev).double()[None, :, None, None] * theta
    cos, sin = m * phi.cos(), m * phi.sin()
    a, c = ((leaf[..., 0:rot:2], leaf[..., 1:rot:2]) if interleaved
            else (leaf[..., :rot // 2], leaf[..., rot // 2:rot]))
    loss = ((a * cos - c * sin) * (g[..., 0:rot:2] if interleaved else g[..., :rot // 2])).sum()
    loss = loss + ((a * sin + c * cos) * (g[..., 1:rot:2] if interleaved else g[..., rot // 2:rot])).sum()
    loss = loss + (leaf[..., rot:] * g[..., rot:]).sum()
    want, = torch.autograd.grad(loss, leaf)
    _, size = rope(host(g), np.broadcast_to(np.arange(s), (b, s)), theta.cpu().numpy(), interleaved, True, m)
    assert_rope(grad, host(want), size, torch.float32, what="autograd")

    picks = torch.randint(0, x.numel(), (40,), generator=gen, device=dev).tolist()
    y0, _ = ops.rope_qk_t(x, None, theta, interleaved=interleaved, magnitude=m)
    for i in picks:
        moved = x.clone()
        moved.view(-1)[i] += 1.0
        step = (moved.view(-1)[i] - x.view(-1)[i]).double().item()
        y1, _ = ops.rope_qk_t(moved, None, theta, interleaved=interleaved, magnitude=m)
        difference = ((y1.double() - y0.double()) * g.double()).sum().item() / step
        # two outputs, each of two roundings of values up to m (|x1| + |x2| + 1) by 2^-22, weighted by |g|
        bound = 4 * 2.0 ** -22 * m * (2 * x.abs().max().item() + 1) * g.abs().max().item()
        assert abs(difference - grad.view(-1)[i].item()) <= bound


def cache_pair(gen, b, capacity, hk, dk, hv, dv, t):
    return make(gen, (b, capacity, hk, dk), t), make(gen, (b, capacity, hv, dv), t)


def expected_caches(k_cache, v_cache, k, v, theta, lengths, counts, positions, interleaved, magnitude=1.0):
    """(K cache, sums of magnitudes, V cache) after the append, in 64 bits."""
    want_k, want_v, size = host(k_cache), host(v_cache), np.zeros(k_cache.shape)
    turned, added = rope(host(k), positions, theta, interleaved, False, magnitude)
    v = host(v)
    for b in range(len(lengths)):
        for s in range(max(0, min(counts[b], k.shape[1]))):
            row = lengths[b] + s
            if 0 <= row < k_cache.shape[1]:
                want_k[b, row], size[b, row], want_v[b, row] = turned[b, s], added[b, s], v[b, s]
    return want_k, size, want_v


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,s,hq,hk,hv,d,rot,dv,capacity", [
    (1, 1, 1, 1, 1, 2, 2, 1, 1), (5, 1, 8, 2, 2, 128, 128, 128, 40), (3, 17, 12, 12, 12, 128, 128, 128, 64),
    (2, 9, 4, 2, 1, 110, 110, 64, 33), (4, 3, 3, 3, 3, 80, 40, 96, 7), (2, 2, 2, 1, 1, 24, 24, 1100, 5),
])
def test_append_matches_definition(ops, dev, dtype, interleaved, b, s, hq, hk, hv, d, rot, dv, capacity):
    gen = torch.Generator(device=dev).manual_seed(b + 10 * s + d)
    t = DTYPES[dtype]
    q, k, v = make(gen, (b, s, hq, d), t), make(gen, (b, s, hk, d), t), make(gen, (b, s, hv, dv), t)
    kc, vc = cache_pair(gen, b, capacity, hk, d, hv, dv, t)
    theta = ops.rope_theta(rot, device=dev)
    lengths = torch.randint(0, capacity - s + 1, (b,), generator=gen, device=dev)
    counts = torch.randint(0, s + 1, (b,), generator=gen, device=dev)
    ln, cn = lengths.tolist(), counts.tolist()
    positions = np.asarray(ln)[:, None] + np.arange(s)
    want_k, size, want_v = expected_caches(kc, vc, k, v, theta.cpu().numpy(), ln, cn, positions, interleaved)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    before_k = kc.clone()
    qo = ops.rope_append_kv_t(q, k, v, theta, kc, vc, lengths, counts=counts, interleaved=interleaved, status=status)
    assert status.item() == 0
    assert_rope(kc, want_k, size, t, capacity * 1.0, "k cache")
    untouched = size.reshape(b, capacity, -1).sum(2) == 0
    assert torch.equal(kc.cpu()[torch.from_numpy(untouched)], before_k.cpu()[torch.from_numpy(untouched)])
    assert np.array_equal(host(vc), want_v)
    want_q, size_q = rope(host(q), positions, theta.cpu().numpy(), interleaved)
    assert_rope(qo, want_q, size_q, t, capacity * 1.0, "q")


def test_append_flags_rows_without_room_and_bad_counts(ops, dev):
    gen = torch.Generator(device=dev).manual_seed(3)
    b, s, h, d, capacity = 5, 4, 2, 16, 6
    q, k, v = (make(gen, (b, s, h, d), torch.float16) for _ in range(3))
    theta = ops.rope_theta(d, device=dev)
    kc, vc = cache_pair(gen, b, capacity, h, d, h, d, torch.float16)
    lengths = torch.tensor([4, -2, 0, 6, 1], device=dev)   # two rows over, two before, -, all over, -
    counts = torch.tensor([4, 4, 4, 4, 4], device=dev)
    positions = lengths.cpu().numpy()[:, None] + np.arange(s)
    want_k, size, want_v = expected_caches(kc, vc, k, v, theta.cpu().numpy(), lengths.tolist(), counts.tolist(),
                                           positions, False)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    ops.rope_append_kv_t(q, k, v, theta, kc, vc, lengths, counts=counts, status=status)
    assert status.item() == ops.APPEND_NO_ROOM
    assert_rope(kc, want_k, size, torch.float16)
    assert np.array_equal(host(vc), want_v)
    status.zero_()
    lengths, counts = torch.zeros(b, dtype=torch.int64, device=dev), torch.tensor([9, -1, 0, 2, 4], device=dev)
    want_k, size, want_v = expected_caches(kc, vc, k, v, theta.cpu().numpy(), lengths.tolist(), counts.tolist(),
                                           np.broadcast_to(np.arange(s), (b, s)), False)
    ops.rope_append_kv_t(q, k, v, theta, kc, vc, lengths, counts=counts, status=status)
    assert status.item() == ops.APPEND_BAD_COUNT
    assert_rope(kc, want_k, size, torch.float16)
    assert np.array_equal(host(vc), want_v)


def test_append_positions_of_their_own_and_strided_caches(ops, dev):
    """Left-padded prompts: positions count from the first real token; the caches lie [batch, heads, capacity, dim]."""
    gen = torch.Generator(device=dev).manual_seed(4)
    b, s, hq, hk, d, capacity = 3, 8, 4, 2, 64, 20
    t = torch.bfloat16
    q, k, v = make(gen, (b, s, hq, d), t), make(gen, (b, s, hk, d), t), make(gen, (b, s, hk, d), t)
    kc = make(gen, (b, hk, capacity, d), t).transpose(1, 2)
    vc = make(gen, (b, hk, capacity, d + 8), t)[..., 8:].transpose(1, 2)
    theta = ops.rope_theta(d, device=dev)
    lengths = torch.tensor([0, 5, 12], device=dev)
    positions = (torch.arange(s) - torch.tensor([[3], [0], [6]])).clamp(min=0).to(dev)
    want_k, size, want_v = expected_caches(kc, vc, k, v, theta.cpu().numpy(), lengths.tolist(), [s] * b,
                                           positions.cpu().numpy(), False, 1.5)
    qo = ops.rope_append_kv_t(q, k, v, theta, kc, vc, lengths, positions=positions, magnitude=1.5)
    assert_rope(kc, want_k, size, t)
    assert np.array_equal(host(vc), want_v)
    want_q, size_q = rope(host(q), positions.cpu().numpy(), theta.cpu().numpy(), False, False, 1.5)
    assert_rope(qo, want_q, size_q, t)


def test_append_past_32_bit_offsets(ops, dev):
    """A cache of 2.2e9 values: rows behind 2^31 elements."""
    b, capacity, h, d = 2, 540000, 16, 128  # 1.1e9 values a sequence
    gen = torch.Generator(device=dev).manual_seed(9)
    kc = torch.zeros((b, capacity, h, d), dtype=torch.float16, device=dev)
    vc = torch.zeros((b, capacity, 1, 8), dtype=torch.float16, device=dev)
    q, k, v = make(gen, (b, 2, 1, d), kc.dtype), make(gen, (b, 2, h, d), kc.dtype), make(gen, (b, 2, 1, 8), kc.dtype)
    theta = ops.rope_theta(d, device=dev)
    lengths = torch.tensor([7, capacity - 2], device=dev)
    ops.rope_append_kv_t(q, k, v, theta, kc, vc, lengths)
    rows = lengths.cpu().numpy()[:, None] + np.arange(2)
    want, size = rope(host(k), rows, theta.cpu().numpy())
    got = torch.stack([kc[i, lengths[i]:lengths[i] + 2] for i in range(b)])
    assert_rope(got, want, size, kc.dtype, float(capacity))
    assert int(torch.count_nonzero(kc)) == int(torch.count_nonzero(got))


def test_append_captured_step_follows_the_lengths(ops, dev):
    """A captured step, replayed while lengths, counts and inputs change, equals eager calls bit for bit; two
    captured graphs share nothing."""
    gen = torch.Generator(device=dev).manual_seed(10)
    b, hq, hk, d, capacity, t = 4, 8, 2, 128, 16, torch.float16
    theta = ops.rope_theta(d, device=dev)
    q, k, v = make(gen, (b, 1, hq, d), t), make(gen, (b, 1, hk, d), t), make(gen, (b, 1, hk, d), t)
    lengths = torch.tensor([0, 3, 1, 9], device=dev)
    start = lengths.clone()
    caches = [cache_pair(gen, b, capacity, hk, d, hk, d, t) for _ in range(2)]
    twins = [(kc.clone(), vc.clone()) for kc, vc in caches]
    outs = [torch.empty_like(q) for _ in range(2)]
    ops.rope_append_kv_t(q, k, v, theta, *[c.clone() for c in caches[0]], lengths)  # loads the kernel
    graphs = []
    for (kc, vc), out in zip(caches, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.rope_append_kv_t(q, k, v, theta, kc, vc, lengths, q_out=out)
        graphs.append(graph)
    for step in range(4):
        fresh = [make(gen, x.shape, t) for x in (q, k, v)]
        for x, y in zip((q, k, v), fresh):
            x.copy_(y)
        for graph, (kc, vc), out, (kt, vt) in zip(graphs, caches, outs, twins):
            graph.replay()
            want = ops.rope_append_kv_t(q, k, v, theta, kt, vt, lengths)
            assert torch.equal(out, want) and torch.equal(kc, kt) and torch.equal(vc, vt)
        lengths += 1
    assert torch.equal(lengths, start + 4)


def test_rope_on_another_stream(ops, dev):
    gen = torch.Generator(device=dev).manual_seed(11)
    q = make(gen, (4, 500, 8, 64), torch.float32)
    theta = ops.rope_theta(64, device=dev)
    want, _ = ops.rope_qk_t(q, None, theta)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream(device=dev)
    with torch.cuda.stream(stream):
        x = q * 1.0
        for _ in range(3):
            got, _ = ops.rope_qk_t(x, None, theta)
    stream.synchronize()
    assert torch.equal(got, want)


def test_rope_on_a_device_that_is_not_current(ops, dev):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    gen = torch.Generator(device=dev).manual_seed(12)
    q = make(gen, (2, 5, 4, 64), torch.float32)
    theta = ops.rope_theta(64, device=dev)
    want, _ = ops.rope_qk_t(q, None, theta)
    other = torch.device("cuda:1")
    got, _ = ops.rope_qk_t(q.to(other), None, theta.to(other))
    assert got.device == other and torch.equal(got.cpu(), want.cpu())
    with pytest.raises(ValueError, match="one CUDA device"):
        ops.rope_qk_t(q, None, theta.to(other))


def test_rope_empty(ops, dev):
    theta = ops.rope_theta(8, device=dev)
    q = torch.empty((2, 0, 4, 8), device=dev)
    assert ops.rope_qk_t(q, q, theta)[0].shape == q.shape
    none = torch.empty((1, 3, 0, 8), device=dev)
    assert ops.rope_qk_t(none, None, theta)[0].shape == none.shape


@pytest.mark.parametrize("seed", range(24))
def test_rope_random_layouts(ops, dev, seed):
    """Shapes, strides, offsets and options drawn at random, so that every vector width is met."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    t = list(DTYPES.values())[seed % 3]
    b, s = int(rng.integers(1, 5)), int(rng.integers(1, 200))
    hq, hk = int(rng.integers(1, 9)), int(rng.integers(1, 5))
    d = int(rng.choice([2, 4, 6, 8, 16, 20, 32, 36, 64, 72, 100, 128, 136, 144, 192]))
    rot = 2 * int(rng.integers(1, d // 2 + 1)) if rng.random() < 0.5 else d

    def tensor(h):
        pad, off = int(rng.choice([0, 0, 1, 2, 4, 8])), int(rng.choice([0, 0, 1, 2, 4, 8]))
        big = make(gen, (b, s, h * (d + pad) + off), t)
        return big[:, :, off:].unflatten(2, (h, d + pad))[..., :d]

    q, k = tensor(hq), tensor(hk)
    positions = torch.randint(-50, 100000, (b, s), generator=gen, device=dev)
    theta = ops.rope_theta(rot, device=dev)
    check_qk(ops, q, k, theta, positions, t, interleaved=bool(seed & 1), adjoint=bool(seed & 2),
             magnitude=float(rng.choice([1.0, 0.9])))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_in_place_in_a_fused_projection(ops, dev, dtype, interleaved):
    """q and k turned where they lie between one another and v; and a step into the free rows between."""
    gen = torch.Generator(device=dev).manual_seed(13)
    t, b, s, hq, hk, d = DTYPES[dtype], 2, 23, 4, 2, 64
    fused = make(gen, (b, s, hq + 2 * hk, d), t)
    before = fused.clone()
    theta = ops.rope_theta(d, device=dev)
    q, k = fused[:, :, :hq], fused[:, :, hq:hq + hk]
    want_q, want_k = ops.rope_qk_t(before[:, :, :hq], before[:, :, hq:hq + hk], theta, start=3, interleaved=interleaved)
    ops.rope_qk_t(q, k, theta, start=3, interleaved=interleaved, q_out=q, k_out=k)
    assert torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(fused[:, :, hq + hk:], before[:, :, hq + hk:])
    rows = make(gen, (b, 2 * s, hq, d), t)
    before = rows.clone()
    ops.rope_qk_t(rows[:, ::2], None, theta, interleaved=interleaved, q_out=rows[:, 1::2])
    assert torch.equal(rows[:, 1::2], ops.rope_qk_t(before[:, ::2], None, theta, interleaved=interleaved)[0])
    assert torch.equal(rows[:, ::2], before[:, ::2])


def test_append_of_a_token_that_lies_in_its_cache(ops, dev):
    """A projection may write a token's k and v to a row of the caches themselves; the append turns k and takes both
    to the sequence's row, which may be that one."""
    gen = torch.Generator(device=dev).manual_seed(14)
    b, h, d, capacity, t = 3, 2, 64, 9, torch.float16
    theta = ops.rope_theta(d, device=dev)
    q = make(gen, (b, 1, h, d), t)
    kc, vc = cache_pair(gen, b, capacity, h, d, h, d, t)
    kt, vt = kc.clone(), vc.clone()
    lengths = torch.tensor([5, 0, 8], device=dev)
    for row in (5, 0, 8):
        got = ops.rope_append_kv_t(q, kc[:, row:row + 1], vc[:, row:row + 1], theta, kc, vc, lengths)
        want = ops.rope_append_kv_t(q, kt[:, row:row + 1].clone(), vt[:, row:row + 1].clone(), theta, kt, vt, lengths)
        assert torch.equal(got, want) and torch.equal(kc, kt) and torch.equal(vc, vt)


def test_rope_refuses_overlapping_views(ops, dev):
    theta = ops.rope_theta(16, device=dev)
    big = torch.zeros((2, 7, 3, 16), device=dev)
    with pytest.raises(ValueError, match="its own input"):
        ops.rope_qk_t(big[:, :-1], None, theta, q_out=big[:, 1:])
    with pytest.raises(ValueError, match="another tensor's"):
        ops.rope_qk_t(torch.zeros((2, 5, 3, 16), device=dev), big[:, :5], theta, q_out=big[:, 2:])
    lengths = torch.zeros(2, dtype=torch.int64, device=dev)
    q = torch.zeros((2, 3, 3, 16), device=dev)
    with pytest.raises(ValueError, match="its own input"):
        ops.rope_append_kv_t(q, big[:, 1:4], q.clone(), theta, big, big.clone(), lengths)
    with pytest.raises(ValueError, match="another tensor's"):
        ops.rope_append_kv_t(q, q, q, theta, big[:, :6], big[:, 1:], lengths)
    assert int(torch.count_nonzero(big)) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("off,d,rot", [(0, 8192, 8192), (0, 8192, 4096), (1, 8192, 8192), (1, 8190, 54), (0, 2056, 1032),
                                       (0, 3000, 3000)])
def test_rope_heads_wider_than_a_block(ops, dev, dtype, interleaved, off, d, rot):
    """More vectors in a head than a CTA has threads: the CTA goes over the head in passes, with the same turns (one
    value an access, 8192 turned: 64 KB of them) and the same staging room."""
    gen = torch.Generator(device=dev).manual_seed(d + rot)
    t = DTYPES[dtype]
    for b, s, hq, hk in ((1, 1, 1, 1), (2, 3, 2, 1)):
        q = make(gen, (b, s, hq * d + off), t)[:, :, off:].unflatten(2, (hq, d))
        k = make(gen, (b, s, hk * d + off), t)[:, :, off:].unflatten(2, (hk, d))
        positions = torch.randint(0, 5000, (b, s), generator=gen, device=dev)
        theta = ops.rope_theta(rot, device=dev)
        check_qk(ops, q, k, theta, positions, t, interleaved=interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,dv", [(16, 8191), (64, 8192), (8192, 8), (4100, 5000)])
def test_append_heads_wider_than_a_block(ops, dev, interleaved, d, dv):
    gen = torch.Generator(device=dev).manual_seed(d + dv)
    b, s, capacity, t = 2, 3, 5, torch.float16
    q, k, v = make(gen, (b, s, 2, d), t), make(gen, (b, s, 1, d), t), make(gen, (b, s, 1, dv), t)
    kc, vc = cache_pair(gen, b, capacity, 1, d, 1, dv, t)
    theta = ops.rope_theta(d, device=dev)
    lengths, counts = torch.tensor([1, 2], device=dev), torch.tensor([3, 2], device=dev)
    positions = np.asarray([[1, 2, 3], [2, 3, 4]])
    want_k, size, want_v = expected_caches(kc, vc, k, v, theta.cpu().numpy(), [1, 2], [3, 2], positions, interleaved)
    qo = ops.rope_append_kv_t(q, k, v, theta, kc, vc, lengths, counts=counts, interleaved=interleaved)
    assert_rope(kc, want_k, size, t, float(capacity), "k cache")
    assert np.array_equal(host(vc), want_v)
    want_q, size_q = rope(host(q), positions, theta.cpu().numpy(), interleaved)
    assert_rope(qo, want_q, size_q, t, float(capacity), "q")
