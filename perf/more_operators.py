"""Three operators of a decode step, each in its plain form and as the
library's call, and the calls their performance is judged by.

  rope     norms of query and key heads, the rotation (one position or several
           axes) and the split of a projection's rows, into dense tensors
           (qk_norm_rope) or with keys and values into a paged cache
           (qk_norm_rope_kv_append_paged);
  attend   decode attention of sequences that share long prefixes, group by
           group (attention_decode_paged_prefix);
  sample   temperature, top-k, top-p, min-p and the draw of a token from given
           random numbers (sample_filtered_batched).

`listed()` holds the fixed cases, `draw(rng)` more of the same ranges;
`prepare` makes a case's inputs on the GPU from a seed, `run` is one pass over
them - the library's call where `own` is true, elementary torch operations
otherwise -, `work` the bytes and operations a pass cannot do without, and
`exact` the outputs in 64 bits, written from the definitions.
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"
EPS = 1e-6


def listed():
    return [
        # rope, a decode step: one token for each of 64 conversations, into
        # the paged cache
        dict(name="rope_step", kind="rope", paged=True, dtype="bf16", t=64, hq=32, hkv=8, d=128,
             rot=128, axes=1, neox=True, norm=True, theta=1e6, far=8192, page=16, pad=0),
        # packed prompts into the paged cache, 16384 tokens, some of padding
        dict(name="rope_prompts", kind="rope", paged=True, dtype="bf16", t=16384, hq=32, hkv=8,
             d=128, rot=128, axes=1, neox=True, norm=True, theta=1e6, far=4096, page=16, pad=200),
        # an image's or a video's tokens: time, height and width
        dict(name="rope_axes", kind="rope", paged=False, dtype="f16", t=6001, hq=16, hkv=2, d=128,
             rot=128, axes=3, neox=True, norm=True, theta=1e6, far=500, page=0, pad=0),
        # float32, interleaved pairs over half of a head of odd size, far
        # positions, rows inside wider ones
        dict(name="rope_f32", kind="rope", paged=False, dtype="f32", t=333, hq=10, hkv=5, d=96,
             rot=48, axes=1, neox=False, norm=True, theta=1e4, far=1000000, page=0, pad=64),
        # attend, the smallest call: four short conversations under one
        # system prompt, where latency and launches are all there is
        dict(name="attend_small", kind="attend", dtype="bf16", hkv=8, group=4, d=64, page=16,
             sizes=1, b=4, plo=500, phi=500, lo=20, hi=200, lens_seed=3),
        # a full batch of conversations of very different length under one
        # long system prompt
        dict(name="attend_chat", kind="attend", dtype="bf16", hkv=8, group=4, d=128, page=16,
             sizes=1, b=64, plo=8192, phi=8192, lo=16, hi=2000, lens_seed=4),
        # five groups with prompts of their own, larger blocks
        dict(name="attend_groups", kind="attend", dtype="f16", hkv=8, group=8, d=128, page=32,
             sizes=5, b=48, plo=1000, phi=16000, lo=0, hi=3001, lens_seed=5),
        # questions about one document of 131071 tokens
        dict(name="attend_long", kind="attend", dtype="bf16", hkv=8, group=4, d=128, page=16,
             sizes=1, b=16, plo=131071, phi=131071, lo=1, hi=500, lens_seed=6),
        # float32, groups of 5 heads, a head of 96, blocks of no power of two
        dict(name="attend_f32", kind="attend", dtype="f32", hkv=4, group=5, d=96, page=24,
             sizes=2, b=7, plo=100, phi=3001, lo=0, hi=700, lens_seed=7),
        # sample, the smallest call: two rows of a small vocabulary
        dict(name="sample_small", kind="sample", dtype="f32", rows=2, n=32000, k=40, p=0.95,
             minp=0.0, temp=0.8, each=False, flat=1.0, pad=0),
        # a full batch over a large vocabulary, each row its own parameters
        dict(name="sample_batch", kind="sample", dtype="f32", rows=64, n=128256, k=200, p=0.9,
             minp=0.05, temp=0.9, each=True, flat=1.0, pad=0),
        # many rows of nearly flat logits in 16 bits (ties), a padded
        # vocabulary
        dict(name="sample_flat", kind="sample", dtype="bf16", rows=301, n=50257, k=0, p=0.98,
             minp=0.0, temp=1.5, each=False, flat=0.2, pad=47),
    ]


def _log(rng, lo, hi):
    """An int in [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "attend", "attend", "attend", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "rope":
        d = rng.choice([64, 80, 96, 128, 128, 256])
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 4, 5, 8])
        paged = rng.random() < 0.5
        most = int(2e8 / ((hq + 2 * hkv) * d * BYTES[dtype]))
        return dict(kind=kind, paged=paged, dtype=dtype, t=_log(rng, 1, min(16384, most)), hq=hq,
                    hkv=hkv, d=d, rot=rng.choice([d, d, d // 2]), axes=rng.choice([1, 1, 2, 3]),
                    neox=rng.random() < 0.6, norm=rng.random() < 0.8,
                    theta=rng.choice([1e4, 5e5, 1e6]), far=_log(rng, 100, 1000000),
                    page=rng.choice([16, 24, 64]) if paged else 0, pad=rng.choice([0, 0, 1, 64]))
    if kind == "attend":
        c = dict(kind=kind, dtype=dtype, hkv=rng.choice([1, 2, 4, 8, 16]),
                 group=rng.choice([1, 2, 4, 5, 8, 16]), d=rng.choice([64, 96, 128, 128]),
                 page=rng.choice([16, 16, 24, 32, 64]), sizes=rng.choice([1, 1, 2, 3, 6]))
        c["b"] = _log(rng, max(2, c["sizes"]), 128)
        # at most 0.3 GB of K and V, and 2e11 operations
        room = 3e8 / (2 * c["hkv"] * c["d"] * BYTES[dtype])
        room = min(room, 2e11 * c["sizes"] / (4 * c["hkv"] * c["group"] * c["d"] * c["b"]))
        if dtype == "f32":
            room /= 8
        phi = _log(rng, 64, max(128, min(131071, int(room / c["sizes"]))))
        hi = _log(rng, 1, max(2, min(4000, int(room / 2 / c["b"]))))
        return dict(c, plo=rng.randint(0, phi), phi=phi, lo=rng.randint(0, hi), hi=hi,
                    lens_seed=rng.randrange(1 << 20))
    n = _log(rng, 1000, 262144)
    return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, min(512, 16000000 // n)), n=n,
                k=rng.choice([0, 0, 1, 20, 50, 1000]), p=rng.choice([1.0, 0.99, 0.95, 0.9, 0.5]),
                minp=rng.choice([0.0, 0.0, 0.02, 0.1]), temp=rng.choice([0.0, 0.6, 1.0, 1.0, 1.7]),
                each=rng.random() < 0.5, flat=rng.choice([0.2, 1.0, 1.0, 2.0]),
                pad=rng.choice([0, 0, 1, 47]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int32), device=DEV)


def _randn(gen, shape, dtype):
    """Normal values of that type; a large tensor is made a part at a time."""
    out = torch.empty(shape, dtype=dtype, device=DEV)
    flat = out.view(-1)
    for lo in range(0, flat.numel(), 1 << 26):
        part = flat[lo:lo + (1 << 26)]
        part.copy_(torch.randn(part.shape, generator=gen, device=DEV))
    return out


def _sections(c):
    """The pairs of each axis: the first a little fewer, as images have it."""
    pairs = c["rot"] // 2
    rest = pairs // c["axes"]
    return [pairs - (c["axes"] - 1) * rest] + [rest] * (c["axes"] - 1)


def _prepare_rope(c, gen):
    t, width = c["t"], (c["hq"] + 2 * c["hkv"]) * c["d"]
    dt = DTYPES[c["dtype"]]
    # rows inside wider ones where there is padding (a fused projection)
    qkv = _randn(gen, (t, width + (0 if c["paged"] else c["pad"])), dt)[:, :width]
    shape = (t,) if c["axes"] == 1 else (c["axes"], t)
    pos = torch.randint(0, c["far"], shape, generator=gen, device=DEV, dtype=torch.int32)
    w = [torch.randn(c["d"], generator=gen, device=DEV) * 0.2 + 1 for _ in range(2)]
    s = dict(qkv=qkv, q_heads=c["hq"], kv_heads=c["hkv"], q_weight=w[0] if c["norm"] else None,
             k_weight=w[1] if c["norm"] else None, positions=pos, theta=c["theta"],
             rotary_dim=c["rot"], neox=c["neox"],
             sections=None if c["axes"] == 1 else _sections(c))
    if c["paged"]:
        # every token a row of its own somewhere in the pool; the last tokens
        # are a padded batch's, with no slot
        blocks = -(-t // c["page"]) + 7
        slots = torch.randperm(blocks * c["page"], generator=gen, device=DEV)[:t].int()
        slots[t - min(c["pad"], t // 2):] = -1
        pools = [_randn(gen, (blocks, c["hkv"], c["page"], c["d"]), dt) for _ in range(2)]
        s.update(k_pool=pools[0], v_pool=pools[1], slots=slots)
    return s


def _lens(c):
    """The case's lengths: of the groups' prefixes, of the sequences, and how
    many sequences each group has."""
    r = random.Random(c["lens_seed"])
    prefix = [r.randint(c["plo"], c["phi"]) for _ in range(c["sizes"])]
    lens = [r.randint(c["lo"], c["hi"]) for _ in range(c["b"])]
    cuts = sorted(r.sample(range(1, c["b"]), c["sizes"] - 1)) if c["sizes"] > 1 else []
    return prefix, lens, [0] + cuts + [c["b"]]


def _prepare_attend(c, gen):
    prefix, lens, offsets = _lens(c)
    page, dt = c["page"], DTYPES[c["dtype"]]
    needs = [-(-n // page) for n in prefix + lens]
    blocks = sum(needs) + 3
    ids = torch.randperm(blocks, generator=gen, device=DEV).int()
    ends = np.cumsum([0] + needs)

    def table(lo, hi):
        out = torch.zeros((hi - lo, max(1, max(needs[lo:hi]))), dtype=torch.int32, device=DEV)
        for i in range(lo, hi):
            out[i - lo, : needs[i]] = ids[ends[i]:ends[i + 1]]
        return out

    pools = [_randn(gen, (blocks, c["hkv"], page, c["d"]), dt) for _ in range(2)]
    q = torch.randn((c["b"], c["hkv"] * c["group"], c["d"]), generator=gen, device=DEV)
    g = len(prefix)
    return dict(q=(2 * q).to(dt), k_pool=pools[0], v_pool=pools[1], prefix_table=table(0, g),
                prefix_lens=_i32(prefix), block_table=table(g, g + len(lens)), lens=_i32(lens),
                group_offsets=_i32(offsets))


def _prepare_sample(c, gen, seed):
    rows, n = c["rows"], c["n"]
    # normal logits of another width in each row, some tokens far ahead
    x = torch.randn((rows, n + c["pad"]), generator=gen, device=DEV)
    x *= c["flat"] * (torch.rand((rows, 1), generator=gen, device=DEV) * 2 + 1)
    ahead = torch.randint(0, n, (rows, 8), generator=gen, device=DEV)
    x.scatter_add_(1, ahead, c["flat"] * 6 * torch.rand((rows, 8), generator=gen, device=DEV))
    s = dict(logits=x.to(DTYPES[c["dtype"]])[:, :n],
             uniforms=torch.rand(rows, generator=gen, device=DEV), temperature=c["temp"],
             top_k=c["k"], top_p=c["p"], min_p=c["minp"])
    if c["each"]:   # the parameters of requests of every kind in one batch
        r = np.random.RandomState(seed)
        f32 = lambda v: torch.as_tensor(np.asarray(v, np.float32), device=DEV)
        s.update(temperature=f32(c["temp"] * r.choice([0.0, 0.5, 1.0, 1.0, 1.4], rows)),
                 top_k=_i32(c["k"] * r.choice([0, 1, 1, 5], rows)),
                 top_p=f32(np.minimum(1.0, c["p"] * r.choice([0.7, 1.0, 1.0, 2.0], rows))),
                 min_p=f32(c["minp"] * r.choice([0.0, 0.5, 1.0], rows)))
    return s


def prepare(case, seed):
    gen = _gen(seed)
    if case["kind"] == "rope":
        s = _prepare_rope(case, gen)
    elif case["kind"] == "attend":
        s = _prepare_attend(case, gen)
    else:
        s = _prepare_sample(case, gen, seed)
    return case["kind"], s, _lens(case)[2] if case["kind"] == "attend" else None


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _rope(qkv, q_heads, kv_heads, q_weight, k_weight, positions, theta, rotary_dim, neox,
          sections, k_pool=None, v_pool=None, slots=None):
    """The heads' RMS norms, the rotation of their first rotary_dim values,
    and the keys and values into the pools' rows where there are any."""
    t, heads = qkv.shape[0], q_heads + 2 * kv_heads
    x = qkv.float().view(t, heads, -1)
    q, k, v = x[:, :q_heads], x[:, q_heads:-kv_heads], x[:, -kv_heads:]
    pairs = rotary_dim // 2
    freq = theta ** (torch.arange(pairs, device=x.device, dtype=torch.float64) * (-2 / rotary_dim))
    if sections is None:
        pos = positions.double()[:, None]
    else:
        axis = torch.arange(len(sections), device=x.device).repeat_interleave(
            torch.tensor(sections, device=x.device), output_size=pairs)
        pos = positions.double()[axis].T
    angle = pos * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, w):
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        head, rest = x[..., :rotary_dim], x[..., rotary_dim:]
        if neox:
            a, b = head[..., :pairs], head[..., pairs:]
        else:
            a, b = head[..., ::2], head[..., 1::2]
        a, b = a * cos - b * sin, b * cos + a * sin
        head = torch.cat([a, b], -1) if neox else torch.stack([a, b], -1).flatten(-2)
        return torch.cat([head, rest], -1).to(qkv.dtype)

    q, k, v = turned(q, q_weight), turned(k, k_weight), v.to(qkv.dtype)
    if slots is None:
        return q, k, v.contiguous()
    blocks, _, page, _ = k_pool.shape
    held = ((slots >= 0) & (slots < blocks * page)).nonzero()[:, 0]
    at = slots.long()[held]
    k_pool[at // page, :, at % page] = k[held]
    v_pool[at // page, :, at % page] = v[held]
    return q, k_pool, v_pool


def _tokens(pool, table):
    """The rows of the table's blocks, [kv heads, tokens, dim] in float32."""
    x = pool[table.long().clamp(0, pool.shape[0] - 1)].float()
    return x.transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])


def _attend(cuts, q, k_pool, v_pool, prefix_table, prefix_lens, block_table, lens, group_offsets):
    """softmax(q . k / sqrt(D)) . v over the tokens of a sequence's group's
    prefix and its own. Each group's prefix is one product for all of its
    heads; the two parts meet by their maxima and sums."""
    (b, hq, d), (nb, hkv, page, _) = q.shape, k_pool.shape
    rows = hq // hkv
    x = q.float().view(b, hkv, rows, d) / math.sqrt(d)

    def part(x, k, v, seen):   # maximum, sum and weighted values
        w = torch.where(seen, x @ k.transpose(-1, -2).contiguous(), -math.inf)
        top = w.amax(-1, keepdim=True).clamp(min=-1e30)
        w = torch.exp(w - top)
        return top, w.sum(-1, keepdim=True), w @ v

    blocks = block_table.long().clamp(0, nb - 1)
    t = torch.arange(block_table.shape[1] * page, device=q.device)
    k = k_pool[blocks].float().transpose(1, 2).reshape(b, hkv, -1, d)
    v = v_pool[blocks].float().transpose(1, 2).reshape(b, hkv, -1, d)
    top, total, out = part(x, k, v, (t < lens[:, None])[:, None, None, :])
    tops, totals, outs = torch.full_like(top, -1e30), torch.zeros_like(total), torch.zeros_like(out)
    # (cuts: the groups' sequences as the host knows them)
    t = torch.arange(prefix_table.shape[1] * page, device=q.device)
    for g in range(prefix_table.shape[0]):
        lo, hi = cuts[g], cuts[g + 1]
        y = x[lo:hi].transpose(0, 1).reshape(hkv, -1, d)
        k, v = _tokens(k_pool, prefix_table[g]), _tokens(v_pool, prefix_table[g])
        got = part(y, k, v, (t < prefix_lens[g])[None, None, :])
        for whole, piece in zip((tops, totals, outs), got):
            whole[lo:hi] = piece.view(hkv, hi - lo, rows, -1).transpose(0, 1)
    most = torch.maximum(top, tops)
    f, g = torch.exp(top - most), torch.exp(tops - most)
    total, out = total * f + totals * g, out * f + outs * g
    return (out / torch.where(total == 0, 1.0, total)).reshape(b, hq, d).to(q.dtype)


def _sample(logits, uniforms, temperature, top_k, top_p, min_p):
    """A token of each row: the first, in the order of the indices, whose
    running sum of kept weights passes u of their sum. Weights are the whole
    numbers rint(2^40 exp((x - max) / T)); kept are the first k by value, of
    them the fewest with p of their sum, of them those of min_p of the
    largest. T = 0 takes the largest logit."""
    rows, n = logits.shape

    def column(v, dtype):
        if not torch.is_tensor(v):
            v = torch.full((rows,), float(np.float32(v)), device=logits.device)
        return v.to(dtype)[:, None]

    f64 = torch.float64
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    temp, p = column(temperature, f64), column(top_p, f64)
    k, least = column(top_k, torch.int64), column(min_p, f64) * 2.0 ** 40
    near = torch.where(x == top, 0.0, (x - top) / torch.where(temp > 0, temp, 1.0))
    w = torch.round(torch.exp(near) * 2.0 ** 40).long()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    ranked = w.gather(1, order)
    at = torch.arange(n, device=x.device)
    k = torch.where(k > 0, k, n)
    ranked = torch.where(at < k, ranked, 0)
    sums = ranked.cumsum(-1)
    want = p * sums[:, -1:].double()
    keep = (sums - ranked).double() < want     # the sum before it is short of p
    keep = torch.where(p < 1, keep, True) & (at < k) & (ranked.double() >= least)
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ranked, 0))
    sums = kept.cumsum(-1)
    total = sums[:, -1:]
    aim = (uniforms.double()[:, None] * total.double()).floor().long()
    aim = torch.minimum(aim, total - 1).clamp(min=0)
    token = (sums <= aim).sum(-1)
    token = torch.where(temp[:, 0] > 0, token, order[:, 0])
    return torch.where(top[:, 0] > -math.inf, token, -1)


def run(state):
    kind, s, cuts = state
    if own:
        import fusedtok_amd as ft
        if kind == "rope":
            if "slots" in s:
                return ft.qk_norm_rope_kv_append_paged(**s, eps=EPS), s["k_pool"], s["v_pool"]
            return ft.qk_norm_rope(**s, eps=EPS)
        if kind == "attend":
            return ft.attention_decode_paged_prefix(**s)
        return ft.sample_filtered_batched(**s)
    if kind == "attend":
        return _attend(cuts, **s)
    return _rope(**s) if kind == "rope" else _sample(**s)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and the results in 64 bits
# ---------------------------------------------------------------------------


def work(case):
    c = case
    if c["kind"] == "rope":
        values = c["t"] * (c["hq"] + 2 * c["hkv"]) * c["d"]
        return {"bytes": 2 * values * BYTES[c["dtype"]] + 4 * c["t"] * (c["axes"] + 1),
                "flops": 10 * values}
    if c["kind"] == "attend":
        prefix, lens, cuts = _lens(c)
        hq = c["hkv"] * c["group"]
        shared = sum(p * (cuts[g + 1] - cuts[g]) for g, p in enumerate(prefix))
        tokens = sum(prefix) + sum(lens)
        return {"bytes": BYTES[c["dtype"]] * (2 * tokens * c["hkv"] * c["d"] +
                                              2 * c["b"] * hq * c["d"]) + 4 * tokens // c["page"],
                "flops": 4 * (shared + sum(lens)) * hq * c["d"]}
    return {"bytes": c["rows"] * (c["n"] * BYTES[c["dtype"]] + 28), "flops": 20 * c["rows"] * c["n"]}


def _exact_rope(c, s):
    t, d, hq, hkv, rot = c["t"], c["d"], c["hq"], c["hkv"], c["rot"]
    x = s["qkv"].double().reshape(t, hq + 2 * hkv, d)
    pos = s["positions"].double().reshape(c["axes"], t)
    out = x.clone()
    if c["norm"]:
        for lo, hi, w in ((0, hq, s["q_weight"]), (hq, hq + hkv, s["k_weight"])):
            part = x[:, lo:hi]
            out[:, lo:hi] = part / (part.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
    axis = [a for a, m in enumerate(_sections(c)) for _ in range(m)]
    turned = out.clone()
    for j in range(rot // 2):
        i, k = (j, j + rot // 2) if c["neox"] else (2 * j, 2 * j + 1)
        angle = pos[axis[j]] * c["theta"] ** (-2.0 * j / rot)
        co, si = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        turned[:, : hq + hkv, i] = out[:, : hq + hkv, i] * co - out[:, : hq + hkv, k] * si
        turned[:, : hq + hkv, k] = out[:, : hq + hkv, i] * si + out[:, : hq + hkv, k] * co
    q, k, v = turned.split([hq, hkv, hkv], 1)
    if not c["paged"]:
        return q.contiguous(), k.contiguous(), v.contiguous()
    pools = []
    for pool, new in ((s["k_pool"], k), (s["v_pool"], v)):
        flat = pool.double().transpose(1, 2).reshape(-1, hkv, d)   # a row for each slot
        some = s["slots"] >= 0
        flat[s["slots"][some].long()] = new[some]
        pools.append(flat.view(-1, c["page"], hkv, d).transpose(1, 2).contiguous())
    return (q.contiguous(),) + tuple(pools)


def _exact_attend(c, s):
    prefix, lens, cuts = _lens(c)
    hkv, group, d, page = c["hkv"], c["group"], c["d"], c["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)

    def rows(pool, table, n, head):
        ids = table[: -(-n // page)].long()
        return pool[ids, head].double().reshape(-1, d)[:n]

    for g, p in enumerate(prefix):
        for h in range(hkv):
            shared = [rows(pool, s["prefix_table"][g], p, h) for pool in (s["k_pool"], s["v_pool"])]
            for b in range(cuts[g], cuts[g + 1]):
                if p + lens[b] == 0:
                    continue
                k, v = (torch.cat([a, rows(pool, s["block_table"][b], lens[b], h)])
                        for a, pool in zip(shared, (s["k_pool"], s["v_pool"])))
                y = s["q"][b, h * group:(h + 1) * group].double()
                w = torch.softmax(torch.mm(y, k.T.contiguous()) / d ** 0.5, dim=-1)
                out[b, h * group:(h + 1) * group] = torch.mm(w, v)
    return out


def _exact_sample(c, s):
    x = s["logits"].double().cpu().numpy()
    rows, n = x.shape

    def each(v, dtype):
        if torch.is_tensor(v):
            return v.cpu().numpy().astype(dtype)
        return np.full(rows, np.float32(v)).astype(dtype)

    temp, p = each(s["temperature"], np.float64), each(s["top_p"], np.float64)
    k, least = each(s["top_k"], np.int64), each(s["min_p"], np.float64)
    u = s["uniforms"].double().cpu().numpy()
    out = np.zeros(rows, np.int64)
    for r in range(rows):
        if temp[r] <= 0:
            out[r] = int(np.argmax(x[r]))
            continue
        w = np.rint(np.exp((x[r] - x[r].max()) / temp[r]) * 2.0 ** 40).astype(np.int64)
        order = np.lexsort((np.arange(n), -x[r]))
        if k[r] > 0:
            order = order[: k[r]]
        if p[r] < 1:
            sums = np.cumsum(w[order])
            order = order[: 1 + int(np.searchsorted(sums.astype(np.float64), p[r] * float(sums[-1])))]
        order = np.sort(order[(w[order] >= least[r] * 2.0 ** 40)])
        sums = np.cumsum(w[order])
        aim = min(int(u[r] * float(sums[-1])), int(sums[-1]) - 1)
        out[r] = order[int(np.searchsorted(sums, aim, side="right"))]
    return out


def exact(case, seed):
    kind, s, _ = prepare(case, seed)
    if kind == "rope":
        return _exact_rope(case, s)
    if kind == "attend":
        return _exact_attend(case, s)
    return _exact_sample(case, s)
