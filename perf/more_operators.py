"""Timed cases of what several answers from one prompt need: copied pages, attention over a shared prompt, and the
tokens' log probabilities.

* ``copy``   pages of all layers' pools onto others: the last, part-filled page of a forked sequence, or all that is
             held into another pool (``copy_paged``);
* ``shared`` attention of one new token a row, where the rows of a group continue one prompt whose pages they share
             (``decode_attn_shared``);
* ``score``  log probabilities of given tokens, with the entropy and the likeliest alternatives (``token_logprobs``).

Sizes: the head counts, layer counts and vocabularies of the benchmark configurations (12/2, 28/4 and 40/8 query / KV heads of
128, 28 layers or a part of 48, 151936 and 152064 tokens), generic vocabularies, prompts from a short question to 32k tokens,
2 to 64 continuations.  K ~ N(0, 1) with 4 channels per head scaled x20, V and q ~ N(0, 1), as the benchmark draws them.
"""
import math

import torch

own = False

D = 128
DEV = "cuda"
HEADS = ((12, 2), (28, 4), (40, 8))
SM = 1.0 / math.sqrt(D)


def listed():
    return [
        # a chat is forked into four answers: three copies of its last page in every layer
        dict(name="copy_fork", op="copy", dtype="float16", int8=0, layers=28, kv_heads=2, page=16, pages=96, pairs=3,
             slots=13, other=False),
        # a wide fork of an INT8 cache, the layers of a quarter of a model: the prompt's last page for 31 more rows
        dict(name="copy_fork_int8", op="copy", dtype="float16", int8=32, layers=12, kv_heads=8, page=64, pages=64,
             pairs=31, slots=37, other=False),
        # what is held of a pool that has grown moves into a smaller one
        dict(name="copy_compact", op="copy", dtype="bfloat16", int8=0, layers=4, kv_heads=4, page=64, pages=1400,
             pairs=1000, slots=0, other=True),
        # two answers to a short question: latency of a call
        dict(name="shared_short", op="shared", dtype="float16", int8=0, groups=1, rows=2, q_heads=12, kv_heads=2,
             prompt=517, tail=61, page=16),
        # sixteen samples of one long prompt
        dict(name="shared_samples", op="shared", dtype="bfloat16", int8=0, groups=1, rows=16, q_heads=28, kv_heads=4,
             prompt=8191, tail=700, page=16),
        # four prompts of uneven lengths with eight beams each
        dict(name="shared_groups", op="shared", dtype="float16", int8=0, groups=4, rows=8, q_heads=28, kv_heads=4,
             prompt=16384, tail=333, page=32),
        # a long document asked 32 questions, INT8 pages
        dict(name="shared_int8", op="shared", dtype="float16", int8=32, groups=1, rows=32, q_heads=40, kv_heads=8,
             prompt=32768, tail=509, page=64),
        # one decode step's token with five alternatives
        dict(name="score_token", op="score", dtype="float16", rows=1, vocab=32000, top=5, masked=False),
        # a decode step of a batch, with twenty alternatives
        dict(name="score_step", op="score", dtype="bfloat16", rows=32, vocab=151936, top=20, masked=False),
        # a step under a grammar that allows few tokens; rows that no vector load divides
        dict(name="score_masked", op="score", dtype="float32", rows=77, vocab=50257, top=5, masked=True),
        # every token of a prompt scored
        dict(name="score_prompt", op="score", dtype="bfloat16", rows=2047, vocab=152064, top=1, masked=False),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("copy", "shared", "shared", "shared", "score", "score"))
    q_heads, kv_heads = rng.choice(HEADS)
    dtype = rng.choice(("float16", "bfloat16"))
    if op == "score":
        vocab = rng.choice((_log_uniform(rng, 1000, 160000), 32000, 151936, 152064))
        return dict(op=op, dtype=rng.choice((dtype, "float32")), rows=_log_uniform(rng, 1, min(2047, (1 << 28) // vocab)),
                    vocab=vocab, top=rng.choice((0, 1, 2, 5, 10, 20, 32)), masked=rng.random() < 0.25)
    page, int8 = rng.choice((16, 32, 64, 128)), rng.choice((0, 0, 32, 64, 128))
    if op == "copy":
        layers = rng.choice((1, 2, 4, 12) if int8 else (1, 2, 4, 28))
        most = (1 << 29) // (512 * kv_heads * page * layers)  # pages of the pools
        pairs = _log_uniform(rng, 1, min(1000, most // 3))
        return dict(op=op, dtype=dtype, int8=int8, layers=layers, kv_heads=kv_heads, page=page,
                    pages=min(most, 2 * pairs + _log_uniform(rng, 1, 200)), pairs=pairs,
                    slots=rng.choice((0, rng.randint(1, page))), other=rng.random() < 0.4)
    groups = rng.choice((1, 1, 1, 2, 3, 5))
    rows = _log_uniform(rng, 2, 64 // groups)
    return dict(op=op, dtype=dtype, int8=int8, groups=groups, rows=rows, q_heads=q_heads, kv_heads=kv_heads,
                prompt=_log_uniform(rng, 64, min(32768, (1 << 18) // (groups * kv_heads))),
                tail=_log_uniform(rng, 1, min(2048, (1 << 17) // (groups * rows * kv_heads))), page=page)


# ---------------------------------------------------------------- inputs


def _sizes(case):
    """Rows of each group: every other one is a quarter smaller."""
    return [case["rows"] - (g % 2) * (case["rows"] // 4) for g in range(case["groups"])]


def _prompts(case):
    """Tokens of each group's prompt: from all down to a quarter."""
    n, p = case["groups"], case["prompt"]
    return [p - (3 * p // 4) * g // max(n - 1, 1) for g in range(n)]


def _tails(case, n):
    """Tokens of each of n rows behind its prompt: from all down to an eighth."""
    t = case["tail"]
    return [t - (t - (t + 7) // 8) * i // max(n - 1, 1) for i in range(n)]


def _quantized(x, group):
    """INT8 codes and fp16 scales of rows [..., 128], per (row, group)."""
    g = x.float().unflatten(-1, (D // group, group))
    s = (g.abs().amax(-1).clamp(min=1e-5) / 127).half()
    c = (g / s.float().unsqueeze(-1)).round().clamp(-127, 127)
    return c.flatten(-2).to(torch.int8), s


def _outliers(x):
    """K with 4 channels of each head scaled x20; the heads lie along dimension 1."""
    g = torch.Generator().manual_seed(x.shape[1])
    f = torch.ones(x.shape[1], D)
    f.scatter_(1, torch.rand(f.shape, generator=g).argsort(1)[:, :4], 20.0)
    return x * f.to(device=x.device, dtype=x.dtype).view(1, -1, 1, D)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(1000003 * int(seed) + 57)
    dt = getattr(torch, case["dtype"])

    def randn(*shape, dtype=dt):
        return torch.randn(shape, generator=g, device=DEV, dtype=dtype)

    def perm(n):
        return torch.rand(n, generator=g, device=DEV).argsort()

    st = dict(case=case)
    if case["op"] == "score":
        n, v = case["rows"], case["vocab"]
        # a model's logits: a wide bulk and a few tokens that stand out
        x = randn(n, v, dtype=torch.float32).mul_(2.0)
        likely = torch.randint(v, (n, 24), generator=g, device=DEV)
        # (one that is drawn twice has the larger, whichever a GPU writes first)
        x.scatter_reduce_(1, likely, x.gather(1, likely) + torch.rand(n, 24, generator=g, device=DEV) * 12, "amax")
        if case["masked"]:
            x.masked_fill_(torch.rand(n, v, generator=g, device=DEV) < 0.95, -math.inf)
            x.scatter_reduce_(1, likely, torch.rand(n, 24, generator=g, device=DEV) * 8, "amax", include_self=False)
        # mostly tokens that the model holds for likely, as a text has them
        tokens = torch.where(torch.rand(n, generator=g, device=DEV) < 0.7, likely[:, 0],
                             torch.randint(v, (n,), generator=g, device=DEV))
        return dict(st, logits=x.to(dt), tokens=tokens)
    h, ps = case["kv_heads"], case["page"]

    def pool(pages):
        pairs = []
        for x in (_outliers(randn(pages, h, ps, D)), randn(pages, h, ps, D)):
            pairs.append(_quantized(x, case["int8"]) if case["int8"] else (x, None))
        return pairs[0][0], pairs[1][0], pairs[0][1], pairs[1][1]

    if case["op"] == "copy":
        pairs, other = case["pairs"], case["other"]
        st["pools"] = [x for _ in range(case["layers"]) for x in pool(case["pages"]) if x is not None]
        # into an empty pool of what is held, or onto pages that nobody holds
        order = perm(case["pages"])
        st["into"] = [x.new_zeros((pairs, *x.shape[1:])) for x in st["pools"]] if other else None
        st["src"] = order[:pairs].int()
        st["dst"] = (perm(pairs) if other else order[pairs : 2 * pairs]).int()
        st["lens"] = (torch.randint(1, case["slots"] + 1, (pairs,), generator=g, device=DEV).int() if case["slots"]
                      else None)
        if own:  # a beam search copies pages at every step, always of the same pools
            import llm_kvcache_quantization_amd as kvq

            st["handles"] = [None if x is None else kvq.PagePools(x) for x in (st["pools"], st["into"])]
        return st
    hq, sizes, prompts = case["q_heads"], _sizes(case), _prompts(case)
    rows = sum(sizes)
    tails = _tails(case, rows)
    tails = [tails[i] for i in perm(rows).tolist()]
    # a prompt's full pages are shared; what is left of it lies in pages of each row's own, as a fork leaves it
    shared = [p // ps * ps for p in prompts]
    of = [i for i, n in enumerate(sizes) for _ in range(n)]
    lens = [prompts[i] + t for i, t in zip(of, tails)]
    cols = max(-(-n // ps) for n in lens)
    need = sum(s // ps for s in shared) + sum(-(-(n - shared[i]) // ps) for i, n in zip(of, lens))
    numbers = perm(need + 3).tolist()
    first = [[numbers.pop() for _ in range(s // ps)] for s in shared]
    table = [first[i] + [numbers.pop() for _ in range(-(-(n - shared[i]) // ps))] for i, n in zip(of, lens)]
    table = [r + [-1] * (cols - len(r)) for r in table]
    k, v, ks, vs = pool(need + 3)
    st.update(k_pages=k, v_pages=v, k_scale=ks, v_scale=vs, q=randn(rows, hq, D), shared=shared, sizes=sizes,
              table=torch.tensor(table, dtype=torch.int32, device=DEV),
              lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    if own:
        import llm_kvcache_quantization_amd as kvq

        st["prefix"] = kvq.SharedPrefix(sizes, shared, hq, h, device=DEV)
    return st


# ---------------------------------------------------------------- the plain forms


def _plain_copy(st):
    into = st["pools"] if st["into"] is None else st["into"]
    src, dst = st["src"].long(), st["dst"].long()
    for x, to in zip(st["pools"], into):
        pages = x[src]
        if st["lens"] is not None:
            here = torch.arange(x.shape[2], device=DEV) < st["lens"].unsqueeze(1)
            pages = torch.where(here[:, None, :, None], pages, to[dst])
        to[dst] = pages
    return into


def _values(pages, scale, numbers):
    """fp32 [.., Hkv, T, 128] of pages [.., n], one after another."""
    x = pages[numbers].float()
    if scale is not None:
        x = x * scale[numbers].float().repeat_interleave(D // scale.shape[-1], dim=-1)
    return x.transpose(-4, -3).flatten(-3, -2)


def _plain_shared(st):
    c = st["case"]
    ps, h = c["page"], c["kv_heads"]
    rep = c["q_heads"] // h
    out, row = [], 0
    for n, p in zip(st["sizes"], st["shared"]):
        q = st["q"][row : row + n].float().view(n, h, rep, D)
        table, lens = st["table"][row : row + n].clamp(min=0).long(), st["lens"][row : row + n]
        k, v = (_values(st[s + "_pages"], st[s + "_scale"], table[0, : p // ps]) for s in "kv")
        kt, vt = (_values(st[s + "_pages"], st[s + "_scale"], table[:, p // ps :]) for s in "kv")
        here = torch.arange(p, p + kt.shape[2], device=DEV) < lens.unsqueeze(1)
        s0 = (q.transpose(0, 1).reshape(h, n * rep, D) @ k.transpose(1, 2).contiguous()).view(h, n, rep, p).transpose(0, 1)
        s1 = (q @ kt.transpose(2, 3).contiguous()).masked_fill(~here[:, None, None], -math.inf)
        s = torch.cat((s0, s1), -1) * SM
        e = (s - s.amax(-1, keepdim=True)).exp()
        e = e / e.sum(-1, keepdim=True)
        o = (e[..., :p].transpose(0, 1).reshape(h, n * rep, p) @ v).view(h, n, rep, D).transpose(0, 1)
        out.append((o + e[..., p:] @ vt).reshape(n, -1, D).to(st["q"].dtype))
        row += n
    return torch.cat(out)


def _plain_score(st):
    k, logits, tokens = st["case"]["top"], st["logits"], st["tokens"]
    x = logits.float()
    m = x.amax(-1, keepdim=True)
    y = x - m
    e = y.exp()
    l = e.sum(-1, keepdim=True)
    log_l = l.log()
    entropy = log_l.squeeze(1) - torch.where(e > 0, y * e, 0.0).sum(-1) / l.squeeze(1)
    chosen = (y.gather(1, tokens.unsqueeze(1)) - log_l).squeeze(1)
    if not k:
        return chosen, entropy
    # distinct whole numbers in the logits' order, the lower index first among equal ones
    bits = (x + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    order = bits * (1 << 18) + (x.shape[1] - 1 - torch.arange(x.shape[1], device=DEV))
    best = order.topk(k, dim=-1).indices
    return chosen, entropy, y.gather(1, best) - log_l, best


# ---------------------------------------------------------------- one pass


def run(st):
    c = st["case"]
    if not own:
        return {"copy": _plain_copy, "shared": _plain_shared, "score": _plain_score}[c["op"]](st)
    import llm_kvcache_quantization_amd as kvq

    if c["op"] == "copy":
        pools, into = st["handles"]
        kvq.copy_paged(pools, st["src"], st["dst"], st["lens"], into=into)
        return st["pools"] if st["into"] is None else st["into"]
    if c["op"] == "shared":
        return kvq.decode_attn_shared(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lens"], st["prefix"], SM,
                                      k_scale=st["k_scale"], v_scale=st["v_scale"])
    out = kvq.token_logprobs(st["logits"], st["tokens"], c["top"])
    return (out.logprobs, out.entropy) + ((out.top_logprobs, out.top_tokens) if c["top"] else ())


def work(case):
    if case["op"] == "score":
        n, v = case["rows"], case["vocab"]
        size = 4 if case["dtype"] == "float32" else 2
        # a logit's difference to the maximum, exponential, two sums and the comparison with the best so far
        return {"bytes": n * (v * size + 16 + 12 * case["top"]), "flops": 6 * n * v}
    h, ps = case["kv_heads"], case["page"]
    cell = 2 * (D + 2 * D // case["int8"]) if case["int8"] else 4 * D  # K and V of a (token, head)
    if case["op"] == "copy":
        slots = (case["slots"] + 1) / 2 if case["slots"] else ps  # on average
        return {"bytes": int(2 * case["pairs"] * case["layers"] * h * slots * cell), "flops": 0}
    sizes, prompts = _sizes(case), _prompts(case)
    shared = [p // ps * ps for p in prompts]
    rest = sum(n * (p - s) for n, p, s in zip(sizes, prompts, shared)) + sum(_tails(case, sum(sizes)))
    pairs = sum(n * s for n, s in zip(sizes, shared)) + rest
    return {"bytes": h * cell * (sum(shared) + rest) + 4 * D * case["q_heads"] * sum(sizes),
            "flops": 4 * D * case["q_heads"] * pairs}


# ---------------------------------------------------------------- in 64 bits


def exact(case, seed):
    """The outputs by the definitions in 64 bits (codes and the alternatives' numbers have no such value)."""
    st = prepare(case, seed)
    if case["op"] == "copy":
        src, dst = st["src"].tolist(), st["dst"].tolist()
        lens = [case["page"]] * len(src) if st["lens"] is None else st["lens"].tolist()
        out = []
        for x, to in zip(st["pools"], st["into"] or st["pools"]):
            out.append(to.double() if to.is_floating_point() else None)
            if out[-1] is not None:
                for full in set(lens):
                    i = [j for j, n in enumerate(lens) if n == full]
                    s, d = ([y[j] for j in i] for y in (src, dst))
                    out[-1][d, :, :full] = x[s, :, :full].double()
        return out
    if case["op"] == "score":
        rows = []
        for x, t in zip(st["logits"].split(64), st["tokens"].split(64)):
            lp = torch.log_softmax(x.double(), 1)
            p = lp.exp()
            part = [lp.gather(1, t[:, None])[:, 0], -(p * lp).nan_to_num(nan=0.0).sum(1)]
            if case["top"]:
                part.append(lp.sort(1, descending=True).values[:, : case["top"]])
            rows.append(part)
        out = [torch.cat(p) for p in zip(*rows)]
        return tuple(out + [None]) if case["top"] else tuple(out)
    q = st["q"].double()
    out = torch.zeros_like(q)
    rep = case["q_heads"] // case["kv_heads"]
    for b, n in enumerate(st["lens"].tolist()):
        t = torch.arange(n, device=DEV)
        page, slot = st["table"][b, t // case["page"]].long(), t % case["page"]
        for h in range(case["kv_heads"]):
            kv = []
            for x, s in ((st["k_pages"], st["k_scale"]), (st["v_pages"], st["v_scale"])):
                x = x[page, h, slot].double()
                if s is not None:
                    x = (x.view(n, -1, case["int8"]) * s[page, h, slot].double()[..., None]).view(n, D)
                kv.append(x)
            p = torch.softmax(torch.mm(q[b, h * rep : (h + 1) * rep], kv[0].t().contiguous()) * SM, 1)
            out[b, h * rep : (h + 1) * rep] = torch.mm(p, kv[1])
    return out
