"""The token-step operators together, as a small guided decoder uses them: add + RMSNorm, rotary positions with the
append to the KV cache, attention over the caches (torch), the CFG combine of two rows' logits, sampling."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from conftest import assert_close
from token_step_reference import assert_rope, host, logprob_tolerance, penalised, rope, sample_row

pytestmark = pytest.mark.gpu


def test_guided_decoding_steps(ops, dev):
    """Three songs decoded for some steps after ragged prompts.  Each operator's outputs are checked against the
    64-bit definition of what it was given, and the caches at the end against all that went into them."""
    gen = torch.Generator(device=dev).manual_seed(0)
    songs, heads, dim, vocab, capacity, prompt, steps = 3, 4, 32, 1000, 24, 9, 6
    width, rows = heads * dim, 2 * songs  # a conditional and an unconditional row of each song

    def weight(*shape):
        return torch.randn(shape, generator=gen, device=dev) / shape[0] ** 0.5

    embed, w_qkv, w_out, w_head = weight(vocab, width) * vocab ** 0.5, weight(width, 3 * width), weight(width, width), \
        3 * weight(width, vocab)
    gamma = 1 + 0.1 * torch.randn(width, generator=gen, device=dev)
    theta = ops.rope_theta(dim, device=dev)
    th = theta.cpu().numpy()
    k_cache = torch.zeros((rows, capacity, heads, dim), device=dev)
    v_cache = torch.zeros_like(k_cache)
    held_k, held_v = np.zeros(k_cache.shape), np.zeros(v_cache.shape)
    sizes = np.zeros(k_cache.shape)
    lengths = torch.zeros(rows, dtype=torch.int64, device=dev)
    counts = torch.tensor([9, 9, 4, 4, 1, 1], device=dev)
    tokens = torch.randint(0, vocab, (rows, prompt), generator=gen, device=dev)
    recent = torch.full((songs, 4), -1, dtype=torch.int64, device=dev)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    for step in range(steps):
        s = tokens.shape[1]
        residual = embed[tokens].reshape(rows * s, width)
        h, y = ops.add_rmsnorm_t(torch.zeros_like(residual), residual, gamma, 1e-5)
        assert torch.equal(h, residual)
        norm = host(residual) / np.sqrt(np.mean(host(residual) ** 2, axis=1, keepdims=True) + 1e-5) * host(gamma)
        assert_close(host(y), norm, 1e-5, "norm")
        qkv = (y @ w_qkv).view(rows, s, 3 * heads, dim)
        q, k, v = qkv.split(heads, dim=2)
        at = lengths.cpu().numpy()[:, None] + np.arange(s)
        n = [s] * rows if counts is None else counts.tolist()
        turned, size = rope(host(k), at, th)
        for r in range(rows):
            held_k[r, at[r, :n[r]]], sizes[r, at[r, :n[r]]] = turned[r, :n[r]], size[r, :n[r]]
            held_v[r, at[r, :n[r]]] = host(v)[r, :n[r]]
        q = ops.rope_append_kv_t(q, k, v, theta, k_cache, v_cache, lengths, counts=counts, status=status)
        want_q, size_q = rope(host(qkv[:, :, :heads]), at, th)
        assert_rope(q, want_q, size_q, torch.float32, float(capacity))
        reach = lengths[:, None] + torch.arange(s, device=dev)
        scores = torch.einsum("bshd,bchd->bhsc", q, k_cache) / dim ** 0.5
        unseen = torch.arange(capacity, device=dev) > reach[:, :, None]
        mixed = torch.einsum("bhsc,bchd->bshd", scores.masked_fill(unseen[:, None], -torch.inf).softmax(-1), v_cache)
        hidden = mixed.reshape(rows * s, width) @ w_out
        _, y = ops.add_rmsnorm_t(hidden, h, gamma, 1e-5)
        lengths = lengths + (s if counts is None else counts)
        last = (torch.full_like(lengths, s) if counts is None else counts) - 1
        logits = y.view(rows, s, width)[torch.arange(rows, device=dev), last] @ w_head
        guided = ops.cfg_combine_t(logits[1::2].contiguous(), logits[0::2].contiguous(), 1.5)
        u = torch.rand(songs, generator=gen, device=dev)
        logprobs = torch.empty(songs, device=dev)
        chosen = ops.sample_tokens_t(guided, u, temperature=0.9, top_k=50, top_p=0.95, recent=recent, penalty=1.1,
                                     logprobs=logprobs, status=status)
        x = penalised(guided, recent.cpu().numpy(), 1.1)
        for r in range(songs):
            token, logprob, w, total, near = sample_row(x[r], u[r].item(), float(np.float32(0.9)), 50, 0.95)
            assert chosen[r].item() == token, (step, r, near)
            assert abs(logprobs[r].item() - logprob) <= logprob_tolerance(logprob, w, total, vocab)
        recent = torch.cat((recent[:, 1:], chosen[:, None]), 1)
        tokens, counts = chosen.repeat_interleave(2)[:, None], None
    assert status.item() == 0
    assert lengths.tolist() == [9 + 5, 9 + 5, 4 + 5, 4 + 5, 1 + 5, 1 + 5]
    assert_rope(k_cache, held_k, sizes, torch.float32, float(capacity))
    assert np.array_equal(host(v_cache), held_v)
