"""GPU test of a decode step as a server runs it, captured once and replayed:
tables -> head norms, rotation and append -> shared-prefix attention ->
logits -> token, for conversations of two groups with a system prompt each.
Every replay is checked against 64-bit plain forms of what the step read.

The attention's bound is that of its own test, and that of the norms and the
rotation on q and k (a value is off by (D/32 + 14) 2^-24 of its pair's length),
which goes into the scores."""

import numpy as np
import torch
import pytest

import fusedtok_amd as ft
from tests import step_refs as refs

pytestmark = pytest.mark.gpu

DEV = "cuda"
HQ, HKV, D, PAGE, VOCAB = 8, 2, 64, 16, 1500
EPS, THETA = 1e-6, 1e4


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int32), device=DEV)


def np64(t):
    return t.double().cpu().numpy()


def test_a_captured_step():
    rng = np.random.default_rng(12)
    gen = torch.Generator(device=DEV).manual_seed(5)
    sizes, plens = [4, 3], [70, 33]
    b, steps = sum(sizes), 37       # the own tokens cross two blocks
    group = np.repeat([0, 1], sizes)
    offsets = [0, 4, 7]
    width = HQ * D

    def weight(*shape):
        return torch.randn(*shape, generator=gen, device=DEV) / shape[-1] ** 0.5

    embed, w_qkv, w_out = weight(VOCAB, width) * width ** 0.5, weight(
        (HQ + 2 * HKV) * D, width), weight(VOCAB, width) * 6
    qw, kw = (1 + 0.2 * torch.randn(D, generator=gen, device=DEV) for _ in range(2))
    blocks = 60
    kp, vp = (torch.full((blocks, HKV, PAGE, D), float("nan"), device=DEV) for _ in range(2))
    ids = rng.permutation(blocks)
    ptable = np.zeros((2, 5), np.int32)
    ptable[0], ptable[1, :3] = ids[:5], ids[5:8]

    # the prompts: one call for both groups, padded rows behind them
    seq, pos = np.repeat([0, 1], plens), np.concatenate([np.arange(n) for n in plens])
    slots = np.concatenate([ptable[seq, pos // PAGE] * PAGE + pos % PAGE, [-1, -1]])
    prompt = weight(len(seq) + 2, width) * width ** 0.5 @ w_qkv.T
    ft.qk_norm_rope_kv_append_paged(prompt, HQ, HKV, qw, kw, i32(np.concatenate([pos, [0, 0]])),
                                    kp, vp, i32(slots), eps=EPS, theta=THETA, neox=True)
    _, pk, pv = refs.qk_norm_rope(np64(prompt[:-2]), HQ, HKV, np64(qw), np64(kw), pos[None], D,
                                  THETA, EPS, True)
    past = [[(pk[seq == g][i], pv[seq == g][i]) for i in range(plens[g])] for g in group]

    # the state of the loop, on the GPU
    table = torch.full((b, 4), -1, dtype=torch.int32, device=DEV)
    lens, n_free = i32([0] * b), i32([blocks - 8])
    free = i32(ids[8:])
    ones, start = i32([1] * b), i32(np.asarray(plens)[group])
    pt, pl, off = i32(ptable), i32(plens), i32(offsets)
    token = torch.arange(b, device=DEV)
    u = torch.zeros(b, device=DEV)
    temps = torch.tensor([0.0, 1.0, 0.7, 1.3, 1.0, 1.0, 0.9], device=DEV)
    ks, ps = i32([0, 0, 5, 50, 1, 0, 20]), torch.tensor([1, 0.9, 1, 0.95, 1, 0.5, 0.8],
                                                        device=DEV)
    ms = torch.tensor([0, 0, 0, 0.05, 0, 0, 0.1], device=DEV)

    def step():
        slots, pos, _, after, left = ft.block_table_extend(table, lens, ones, free, n_free, PAGE,
                                                           b)
        qkv = embed[token] @ w_qkv.T
        q = ft.qk_norm_rope_kv_append_paged(qkv, HQ, HKV, qw, kw, pos + start, kp, vp, slots,
                                            eps=EPS, theta=THETA, neox=True)
        att = ft.attention_decode_paged_prefix(q, kp, vp, pt, pl, table, after, off)
        logits = att.view(b, -1) @ w_out.T
        new = ft.sample_filtered_batched(logits, u, temperature=temps, top_k=ks, top_p=ps,
                                         min_p=ms)
        lens.copy_(after)
        n_free.copy_(left)
        token.copy_(new)
        return qkv, q, att, logits, new

    kept = [t.clone() for t in (table, lens, n_free, token, kp, vp)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                       # (libraries' own set-up, outside the capture)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for t, was in zip((table, lens, n_free, token, kp, vp), kept):
        t.copy_(was)

    eps = (D / 32 + 14) * 2.0 ** -24
    temp, k, p, m = (t.cpu().numpy() for t in (temps, ks, ps, ms))
    for turn in range(steps):
        u.copy_(torch.as_tensor(rng.random(b).astype(np.float32)))
        graph.replay()
        torch.cuda.synchronize()
        qkv, q, att, logits, new = (t.cpu().numpy() for t in outs)
        at = np.asarray(plens)[group] + turn
        rq, rk, rv = refs.qk_norm_rope(qkv.astype(np.float64), HQ, HKV, np64(qw), np64(kw),
                                       at[None], D, THETA, EPS, True)
        assert np.abs(q - rq).max() <= 2 * eps * np.abs(rq).max()
        assert lens.tolist() == [turn + 1] * b
        for x in range(b):
            past[x].append((rk[x], rv[x]))
            keys, values = (np.stack([c[i] for c in past[x]]) for i in (0, 1))
            for h in range(HQ):
                kk, vv = keys[:, h // 4], values[:, h // 4]
                s = kk @ rq[x, h] / np.sqrt(D)
                w = np.exp(s - s.max())
                w /= w.sum()
                size = (np.abs(kk) @ np.abs(rq[x, h])).max() / np.sqrt(D)
                turned = 2 * eps * (np.abs(rq[x, h]).max() * np.abs(kk).sum(1).max() +
                                    np.abs(kk).max() * np.abs(rq[x, h]).sum()) / np.sqrt(D)
                part = ((D / 16 + 22) * size + len(kk) / 16 + 204) * 2.0 ** -24 + turned
                bound = 2 * part * (w @ np.abs(vv)) + 2.0 ** -24 * np.abs(w @ vv)
                assert (np.abs(att[x, h] - w @ vv) <= bound).all()
            assert new[x] == refs.sample(logits[x], u[x].item(), temp[x], k[x], p[x], m[x])
    assert n_free.tolist() == [blocks - 8 - 3 * b]
