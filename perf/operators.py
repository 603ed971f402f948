"""Serving operators of the decoder for several hypotheses per clip: 8-bit projections, a paged KV cache whose pages
hypotheses share, and the attention that reads a shared prefix once.  Cases, plain forms and calls for measuring them.

  i8        one projection with 8-bit integer weights (a scale per output channel) and activations that are rounded to
            8 bits per token inside the call: y = (q(x) . w^T) * s_x * s_w + bias
  attn      one layer's attention of a step: the step's K / V rows go into the paged cache, then every query row attends to
            its sequence's keys; the sequences of a group (the hypotheses of one clip) share the pages of their prefix
  fork      hypotheses of every clip start from its prompt: their page tables are forked and room for the next tokens is
            made, which copies the prompt's last, partly filled page for each of them
  turnover  clips leave and others come, twice: pages are freed, the pool is compacted, pages are taken again
"""
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_kept = {}


def _i8(name, rows, cols, inner, x="bf16", out="bf16", bias=False, pad=0):
    return dict(name=name, kind="i8", rows=rows, cols=cols, inner=inner, x=x, out=out, bias=bias, pad=pad)


def _attn(name, groups, hyps, shared, own_lo, own_hi, tokens, heads, kv_heads, head_dim=128, page=16):
    return dict(name=name, kind="attn", groups=groups, hyps=hyps, shared=shared, own_lo=own_lo, own_hi=own_hi, tokens=tokens,
                heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page)


def _fork(name, clips, hyps, lo, hi, tokens, layers, kv_heads=8, head_dim=128, page=16):
    return dict(name=name, kind="fork", clips=clips, hyps=hyps, lo=lo, hi=hi, tokens=tokens, layers=layers, kv_heads=kv_heads,
                head_dim=head_dim, page=page)


def _turnover(name, first, second, lo, hi, layers, kv_heads=8, head_dim=128, page=16):
    return dict(name=name, kind="turnover", first=first, second=second, lo=lo, hi=hi, layers=layers, kv_heads=kv_heads,
                head_dim=head_dim, page=page)


def listed():
    return [
        # q/k/v projection of the 1.7B decoder for the one row of a realtime clip's decode step
        _i8("i8 1 x 2048 -> 4096", 1, 4096, 2048),
        # down projection for five hypotheses of one clip
        _i8("i8 5 x 6144 -> 2048", 5, 2048, 6144),
        # a ragged batch against an odd output width and an inner size that ends inside a vector; fp32 rows in and out
        _i8("i8 387 x 1003 -> 1027 f32", 387, 1027, 1003, x="f32", out="f32", bias=True, pad=5),
        # gate/up projection in the prefill of twenty clips of 30 s
        _i8("i8 8100 x 2048 -> 12288", 8100, 12288, 2048),
        # the first step of four hypotheses of one 30 s clip (405 prompt rows)
        _attn("attn 1x4 after 405", 1, 4, 405, 1, 1, 1, 16, 8),
        # a decode step of a serving batch: 96 clips, five hypotheses each, anywhere between their first and last token
        _attn("attn 96x5 after 405", 96, 5, 405, 1, 448, 1, 16, 8),
        # a long shared context (many joined segments) with short answers, eight hypotheses for each of sixteen recordings
        _attn("attn 16x8 after 16000", 16, 8, 16000, 3, 61, 1, 16, 8),
        # scoring given texts: several rows per hypothesis at once, the encoder's head width, no grouped heads, large pages
        _attn("attn 12x7 after 1111 score", 12, 7, 1111, 24, 130, 24, 14, 14, head_dim=64, page=64),
        # five hypotheses of one clip leave its prompt
        _fork("fork 1x5", 1, 5, 405, 405, 1, 28),
        # the hypotheses of a serving batch leave their prompts
        _fork("fork 40x5", 40, 5, 21, 405, 7, 28),
        # two clips against three
        _turnover("turnover 2/3", 2, 3, 100, 420, 28),
        # half of a serving batch ends, then the other half
        _turnover("turnover 16/12", 16, 12, 90, 853, 28),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _drawn(rng):
    kind = rng.choice(("i8", "i8", "attn", "attn", "fork", "turnover"))
    if kind == "i8":
        return _i8("", _log(rng, 1, 9000), _log(rng, 64, 12288), _log(rng, 33, 6144), x=rng.choice(("bf16", "bf16", "f32")),
                   out=rng.choice(("bf16", "bf16", "f32")), bias=rng.random() < 0.5, pad=rng.choice((0, 0, 1, 8, 24)))
    if kind == "attn":
        kv = rng.choice((1, 2, 4, 8, 14))
        own_lo = _log(rng, 1, 100)
        tokens = rng.choice((1, 1, 1, rng.randint(2, 24)))
        return _attn("", _log(rng, 1, 96), rng.randint(1, 16), _log(rng, 1, 16000), max(own_lo, tokens), max(own_lo, tokens) + _log(rng, 1, 448),
                     tokens, kv * rng.choice((1, 2, 4)), kv, head_dim=rng.choice((64, 128)), page=rng.choice((16, 32, 64)))
    layers, kv, dim, page = rng.randint(2, 28), rng.choice((2, 4, 8)), rng.choice((64, 128)), rng.choice((16, 32, 64))
    lo = _log(rng, 1, 400)
    if kind == "fork":
        return _fork("", _log(rng, 1, 80), rng.randint(1, 8), lo, lo + _log(rng, 1, 450), _log(rng, 1, 40), layers, kv, dim, page)
    return _turnover("", _log(rng, 1, 24), _log(rng, 1, 24), lo, lo + _log(rng, 1, 450), layers, kv, dim, page)


def draw(rng):
    cost = {}
    for c in listed():
        w = work(c)
        k = cost.setdefault(c["kind"], {"bytes": 0, "flops": 0})
        cost[c["kind"]] = {n: max(k[n], w[n]) for n in k}
    while True:
        c = _drawn(rng)
        w = work(c)
        if all(w[n] <= cost[c["kind"]][n] for n in w) and _pool_values(c) <= 450_000_000 and _unshared(c) <= 4_500_000_000:
            del c["name"]
            return c


# ---- sizes that follow from a case alone ----

def _spread(lo, hi, n):
    """n whole numbers from lo to hi in equal steps."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)] if n > 1 else [hi]


def _ceil(a, b):
    return -(-a // b)


def _attn_sizes(c):
    """Prefix of every group, own length of every sequence (in the order of a seed), rows of every sequence."""
    shared = _spread(_ceil(c["shared"], 2), c["shared"], c["groups"])
    n = c["groups"] * c["hyps"]
    return shared, _spread(c["own_lo"], c["own_hi"], n), [1 + (7 * i) % c["tokens"] for i in range(n)]


def _pages_needed(c):
    pg = c["page"]
    if c["kind"] == "attn":
        shared, mine, _ = _attn_sizes(c)
        return sum(_ceil(s, pg) + 1 for s in shared) + sum(_ceil(o, pg) + 1 for o in mine)
    if c["kind"] == "fork":
        lens = _spread(c["lo"], c["hi"], c["clips"])
        return sum(_ceil(n, pg) for n in lens) + c["clips"] * c["hyps"] * (1 + _ceil(c["tokens"], pg))
    return sum(_ceil(n, pg) for k in ("first", "second") for n in _spread(c["lo"], c["hi"], c[k]))


def _pool_pages(c):
    return _pages_needed(c) + _pages_needed(c) // 8 + 3


def _pool_values(c):
    return 0 if c["kind"] == "i8" else c.get("layers", 1) * _pool_pages(c) * c["kv_heads"] * c["page"] * c["head_dim"]


def _unshared(c):
    """K values of a pass when every sequence has its own copy of the prefix."""
    return c["groups"] * c["hyps"] * (c["shared"] + c["own_hi"]) * c["kv_heads"] * c["head_dim"] if c["kind"] == "attn" else 0


def work(case):
    c = case
    size = {"bf16": 2, "f32": 4}
    if c["kind"] == "i8":
        m, n, k = c["rows"], c["cols"], c["inner"]
        return {"bytes": m * k * size[c["x"]] + n * k + 4 * n * (2 if c["bias"] else 1) + m * n * size[c["out"]], "flops": 2 * m * n * k}
    token = 2 * 2 * c["kv_heads"] * c["head_dim"]  # K and V of one token and layer
    if c["kind"] == "attn":
        shared, mine, rows = _attn_sizes(c)
        keys = sum(shared) + sum(mine)
        pairs = sum(r * (shared[i // c["hyps"]] + o) for i, (o, r) in enumerate(zip(mine, rows)))
        return {"bytes": keys * token + 2 * sum(rows) * token // 2 + 2 * 2 * sum(rows) * c["heads"] * c["head_dim"],
                "flops": 4 * pairs * c["heads"] * c["head_dim"]}
    pg = c["page"]
    if c["kind"] == "fork":
        lens = _spread(c["lo"], c["hi"], c["clips"])
        tables = sum(_ceil(n + c["tokens"], pg) for n in lens) * c["hyps"]
        return {"bytes": 2 * c["hyps"] * sum(n % pg for n in lens) * token * c["layers"] + 4 * 3 * tables, "flops": 0}
    a, b = (sum(_ceil(n, pg) for n in _spread(c["lo"], c["hi"], c[k])) for k in ("first", "second"))
    return {"bytes": 2 * (2 * min(a, b) * pg * token * c["layers"]) + 4 * 6 * (a + b), "flops": 0}


# ---- what a program has in hand ----

def _model():
    if "model" not in _kept:
        sys.path.insert(0, os.path.join(_ROOT, "qwen3-asr-swift_amd"))
        import q3asr
        _kept["model"] = q3asr.Qwen3ASRModel(q3asr.make_config("tiny"))
        _kept["q3asr"] = q3asr
        _kept["stream"] = torch.cuda.Stream()
    return _kept["q3asr"], _kept["model"], _kept["stream"].cuda_stream


def _ints(v, dev):
    return torch.tensor(np.asarray(v, dtype=np.int32), device=dev)


def _pool(s, c, dev, g):
    shape = (c.get("layers", 1), _pool_pages(c), c["kv_heads"], c["page"], c["head_dim"])
    for n in "kv":
        s[n] = torch.empty(shape, dtype=torch.bfloat16, device=dev).normal_(generator=g)


def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev).manual_seed(int(seed))
    r = np.random.RandomState(int(seed) % (1 << 31))
    s = {"case": dict(case)}
    c = case
    if c["kind"] == "i8":
        m, n, k, ld = c["rows"], c["cols"], c["inner"], c["inner"] + c["pad"]
        # activations after a norm: about unit variance, a few channels far larger, and rows of differing size
        x = torch.randn(m, ld, device=dev, generator=g)
        x *= torch.where(torch.rand(ld, device=dev, generator=g) < 0.01, 12.0, 1.0) * torch.exp(torch.randn(m, 1, device=dev, generator=g) / 2)
        s["x"] = x.to(_DT[c["x"]])[:, :k]
        w = torch.randn(n, k, device=dev, generator=g) * k ** -0.5
        scale = w.abs().amax(1) / 127
        ldw = _ceil(k, 16) * 16
        s["w"] = torch.zeros(n, ldw, dtype=torch.int8, device=dev)[:, :k]
        s["w"].copy_(torch.round(w / scale[:, None]).clamp_(-127, 127))
        s["w_scales"] = scale
        s["bias"] = torch.randn(n, device=dev, generator=g) if c["bias"] else None
        s["out"] = torch.empty(m, n, dtype=_DT[c["out"]], device=dev)
        if own:
            q3, model, s["stream"] = _model()
            s["linear"] = q3.Int8Linear(model, s["w"].data_ptr(), s["w_scales"].data_ptr(), n, k, ldw=ldw,
                                        bias=s["bias"].data_ptr() if c["bias"] else None)
            s["ws"] = torch.empty(s["linear"].workspace_bytes(m), dtype=torch.uint8, device=dev)
        return s
    pages, pg = _pool_pages(c), c["page"]
    _pool(s, c, dev, g)
    order = list(map(int, r.permutation(pages)))  # pages in use lie anywhere in the pool
    if c["kind"] == "attn":
        shared, mine, rows = _attn_sizes(c)
        mine = [mine[i] for i in r.permutation(len(mine))]
        shared = [shared[i] for i in r.permutation(len(shared))]
        lens = [shared[i // c["hyps"]] + o for i, o in enumerate(mine)]
        tables, prefix = [], []
        for i, n in enumerate(lens):
            if i % c["hyps"] == 0:
                prefix = [order.pop() for _ in range(shared[i // c["hyps"]] // pg)]
            tables.append(prefix + [order.pop() for _ in range(_ceil(n, pg) - len(prefix))])
        n_seqs = len(lens)
    elif c["kind"] == "fork":
        lens = [int(n) for n in r.permutation(_spread(c["lo"], c["hi"], c["clips"]))]
        tables = [[order.pop() for _ in range(_ceil(n, pg))] for n in lens]
        n_seqs = c["clips"] * (1 + c["hyps"])
    else:
        lens = [int(n) for k in ("first", "second") for n in r.permutation(_spread(c["lo"], c["hi"], c[k]))]
        tables = [[order.pop() for _ in range(_ceil(n, pg))] for n in lens]
        n_seqs = len(lens)
    width = max(_ceil(n + c.get("tokens", 0), pg) for n in lens)
    table, refs = np.full((n_seqs, width), -1, np.int32), np.zeros(pages, np.int32)
    for i, t in enumerate(tables):
        table[i, :len(t)] = t
        refs[t] += 1
    s["table"], s["refs"] = _ints(table, dev), _ints(refs, dev)
    s["lens"] = _ints(lens + [0] * (n_seqs - len(lens)), dev)
    if c["kind"] == "attn":
        s["seqs"] = _ints(r.permutation(c["groups"])[:, None] * c["hyps"] + np.arange(c["hyps"]), dev).reshape(-1)
        s["cu_rows"] = _ints(np.concatenate([[0], np.cumsum(rows)]), dev)
        s["cu_groups"] = _ints(np.arange(c["groups"] + 1) * c["hyps"], dev)
        s["shared"] = _ints([shared[int(i) // c["hyps"]] // pg * pg for i in s["seqs"][::c["hyps"]].tolist()], dev)
        m, kv = sum(rows), c["kv_heads"] * c["head_dim"]
        # queries and keys as after their norms: unit variance, so that a row's softmax is neither flat nor one key's
        for n, width in (("q", c["heads"] * c["head_dim"]), ("k_rows", kv), ("v_rows", kv)):
            s[n] = torch.randn(m, width, device=dev, generator=g).to(torch.bfloat16)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(m, c["heads"], dtype=torch.float32, device=dev)
    elif c["kind"] == "fork":
        hyps = np.arange(c["clips"] * c["hyps"])
        s["dst"], s["src"] = _ints(c["clips"] + hyps, dev), _ints(hyps // c["hyps"], dev)
        s["tokens"] = torch.full_like(s["dst"], c["tokens"])
    else:
        cut = c["first"]
        s["sets"] = [(_ints(np.arange(a, b), dev), _ints(lens[a:b], dev)) for a, b in ((0, cut), (cut, len(lens)))]
    if own:
        q3, model, s["stream"] = _model()
        s["status"] = torch.zeros(4, dtype=torch.int32, device=dev)
        s["cache"] = q3.PagedKVCache(model, k=s["k"].data_ptr(), v=s["v"].data_ptr(), layers=c.get("layers", 1), pages=pages,
                                     kv_heads=c["kv_heads"], head_dim=c["head_dim"], page_tokens=pg, table=s["table"].data_ptr(),
                                     lens=s["lens"].data_ptr(), refs=s["refs"].data_ptr(), status=s["status"].data_ptr(),
                                     max_seqs=n_seqs, max_seq_pages=s["table"].shape[1])
        s["ws"] = torch.empty(s["cache"].workspace_bytes(), dtype=torch.uint8, device=dev)
        s["cache"].set_workspace(s["ws"].data_ptr(), s["ws"].numel())
        if c["kind"] == "attn":
            s["batch"] = q3.AttentionBatch(seqs=s["seqs"].data_ptr(), cu_rows=s["cu_rows"].data_ptr(), n=len(lens), rows=sum(rows),
                                           max_rows=max(rows), max_len=max(lens), cu_groups=s["cu_groups"].data_ptr(),
                                           shared=s["shared"].data_ptr(), n_groups=c["groups"],
                                           max_group_rows=max(sum(rows[i:i + c["hyps"]]) for i in range(0, len(rows), c["hyps"])),
                                           max_shared=max(shared) // pg * pg,
                                           max_own=max(n - shared[i // c["hyps"]] // pg * pg for i, n in enumerate(lens)))
            s["attn_ws"] = torch.empty(s["cache"].attention_workspace_bytes(s["batch"], c["heads"]), dtype=torch.uint8, device=dev)
    return s


# ---- plain forms ----

def _plain_i8(s):
    c = s["case"]
    x = s["x"].float()
    scale = (x.abs().amax(1, keepdim=True).double() / 127).float()
    # in 64 bits: a quotient next to the middle of two whole numbers must not be rounded twice
    q = torch.where(scale > 0, torch.round(x.double() / scale.double()), 0.0).clamp(-127, 127).float()
    y = (q @ s["w"].float().T) * scale * s["w_scales"]
    return (y if s["bias"] is None else y + s["bias"]).to(_DT[c["out"]])


def _rows_of(s):
    """Per row of the step: its place in the list of sequences, its number there and its position in the sequence."""
    cu = s["cu_rows"].long()
    r = torch.arange(s["q"].shape[0], device=cu.device)
    i = torch.searchsorted(cu, r, right=True) - 1
    t = r - cu[i]
    return i, t, s["lens"].long()[s["seqs"].long()[i]] - (cu[i + 1] - cu[i]) + t


def _plain_attn(s):
    c = s["case"]
    pg, kv, d, heads = c["page"], c["kv_heads"], c["head_dim"], c["heads"]
    i, t, pos = _rows_of(s)
    table = s["table"].long()[s["seqs"].long()]
    page = table[i, pos // pg]
    s["k"][0, page, :, pos % pg] = s["k_rows"].view(-1, kv, d)
    s["v"][0, page, :, pos % pg] = s["v_rows"].view(-1, kv, d)
    n, width, group, most = table.shape[0], table.shape[1] * pg, heads // kv, int(c["tokens"])
    k, v = (s[x][0][table.clamp(min=0)].permute(0, 2, 1, 3, 4).reshape(n, kv, width, d).float() for x in "kv")
    q = torch.zeros(n, most, heads, d, device=k.device)
    q[i, t] = s["q"].view(-1, heads, d).float()
    q = q.view(n, most, kv, group, d).permute(0, 2, 1, 3, 4).reshape(n, kv, most * group, d)
    place = torch.full((n, most), -1, device=k.device)
    place[i, t] = pos
    seen = torch.arange(width, device=k.device) <= place.repeat_interleave(group, 1)[:, None, :, None]
    score = (q @ k.transpose(2, 3).contiguous() * d ** -0.5).masked_fill_(~seen, float("-inf"))
    top = score.amax(3, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(score - top)
    total = p.sum(3, keepdim=True)
    o = (p @ v) / total.clamp(min=torch.finfo(torch.float32).tiny)
    o = o.view(n, kv, most, group, d).permute(0, 2, 1, 3, 4).reshape(n, most, heads * d)[i, t]
    lse = (top + torch.log(total)).view(n, kv, most, group).permute(0, 2, 1, 3).reshape(n, most, heads)[i, t]
    return {"out": o.to(torch.bfloat16), "lse": lse, "k": s["k"], "v": s["v"]}


def _count(refs, table, by):
    """refs with `by` added for every page that the rows name."""
    flat = table.reshape(-1).long()
    flat = flat[flat >= 0]
    refs.index_add_(0, flat, torch.full_like(flat, by, dtype=refs.dtype))


def _plain_fork(s, dst, src):
    """dst's sequences share the pages of src's; src None: they end."""
    rows = torch.full_like(s["table"][dst], -1) if src is None else s["table"][src]
    lens = torch.zeros_like(s["lens"][dst]) if src is None else s["lens"][src]
    _count(s["refs"], s["table"][dst], -1)
    _count(s["refs"], rows, 1)
    s["table"][dst], s["lens"][dst] = rows, lens


def _plain_reserve(s, seqs, tokens):
    """Room for more tokens. A partly filled page that others hold too is copied first; where all that hold it are in the
    list, the first of them keeps it. Free pages are taken from the lowest on, in the order of the list."""
    pg, refs, table = s["case"]["page"], s["refs"], s["table"]
    n, add = s["lens"][seqs].long(), tokens.long()
    i, fill, last = torch.arange(len(seqs), device=n.device), n % pg, (n - 1).clamp(min=0) // pg
    page = table[seqs, last].long()
    partly = (fill > 0) & (add > 0)
    at = torch.where(partly, page, refs.numel())
    here = torch.zeros(refs.numel() + 1, dtype=torch.long, device=n.device).index_add_(0, at, torch.ones_like(at))
    first = torch.full_like(here, len(seqs)).scatter_reduce_(0, at, i, "amin")
    copy = partly & (refs[page.clamp(min=0)] > 1) & ~((here[at] == refs[page.clamp(min=0)]) & (first[at] == i))
    old, new = (n + pg - 1) // pg, (n + add + pg - 1) // pg
    need = copy.long() + new - old
    start = torch.cumsum(need, 0) - need
    free = torch.nonzero(refs == 0).reshape(-1)[:int(need.sum())]
    for x in "kv":
        src, dst = s[x][:, page[copy]], s[x][:, free[start[copy]]]
        filled = torch.arange(pg, device=n.device) < fill[copy][:, None]
        s[x][:, free[start[copy]]] = torch.where(filled[None, :, None, :, None], src, dst)
    _count(refs, page[copy], -1)
    refs[free] = 1
    table[seqs[copy], last[copy]] = free[start[copy]].to(table.dtype)
    j = torch.arange(table.shape[1], device=n.device)
    more = (j >= old[:, None]) & (j < new[:, None])
    put = free[((start + copy - old)[:, None] + j)[more]].to(table.dtype)
    rows = table[seqs]
    rows[more] = put
    table[seqs] = rows
    s["lens"][seqs] = (n + add).to(s["lens"].dtype)


def _plain_compact(s):
    """Pages in use move to the front of the pool: the lowest of those behind it to its lowest gap, and so on."""
    used = s["refs"] > 0
    n = int(used.sum())
    gaps, far = torch.nonzero(~used[:n]).reshape(-1), torch.nonzero(used[n:]).reshape(-1) + n
    for x in "kv":
        s[x][:, gaps] = s[x][:, far]
    to = torch.arange(used.numel(), device=used.device, dtype=s["table"].dtype)
    to[far] = gaps.to(to.dtype)
    s["refs"][gaps] = s["refs"][far]
    s["refs"][far] = 0
    s["table"].copy_(torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()], -1))


def _state_of(s):
    return {n: s[n] for n in ("table", "lens", "refs", "k", "v")}


def run(state):
    s, c = state, state["case"]
    if c["kind"] == "i8":
        if not own:
            return _plain_i8(s)
        s["linear"](s["x"].data_ptr(), c["rows"], s["out"].data_ptr(), x_dtype=c["x"], ldx=s["x"].stride(0), out_dtype=c["out"],
                    workspace=(s["ws"].data_ptr(), s["ws"].numel()), stream=s["stream"])
        return s["out"]
    if c["kind"] == "attn":
        if not own:
            return _plain_attn(s)
        s["cache"].write(0, s["k_rows"].data_ptr(), s["v_rows"].data_ptr(), s["batch"], stream=s["stream"])
        s["cache"].attention(0, s["q"].data_ptr(), s["out"].data_ptr(), s["batch"], c["heads"], lse=s["lse"].data_ptr(),
                             workspace=(s["attn_ws"].data_ptr(), s["attn_ws"].numel()), stream=s["stream"])
        return {"out": s["out"], "lse": s["lse"], "k": s["k"], "v": s["v"]}
    if c["kind"] == "fork":
        if own:
            s["cache"].fork(s["dst"].data_ptr(), s["src"].data_ptr(), s["dst"].numel(), stream=s["stream"])
            s["cache"].reserve(s["dst"].data_ptr(), s["tokens"].data_ptr(), s["dst"].numel(), stream=s["stream"])
        else:
            _plain_fork(s, s["dst"].long(), s["src"].long())
            _plain_reserve(s, s["dst"].long(), s["tokens"])
        return _state_of(s)
    for seqs, tokens in s["sets"]:
        if own:
            s["cache"].free(seqs.data_ptr(), seqs.numel(), stream=s["stream"])
            s["cache"].compact(stream=s["stream"])
            s["cache"].reserve(seqs.data_ptr(), tokens.data_ptr(), seqs.numel(), stream=s["stream"])
        else:
            _plain_fork(s, seqs.long(), None)
            _plain_compact(s)
            _plain_reserve(s, seqs.long(), tokens)
    return _state_of(s)


# ---- from the definitions, in 64 bits ----

def _exact_attn(s):
    c = s["case"]
    pg, kv, d, heads = c["page"], c["kv_heads"], c["head_dim"], c["heads"]
    group = heads // kv
    cu, lens, table = s["cu_rows"].tolist(), s["lens"].tolist(), s["table"].tolist()
    k_pool, v_pool = s["k"][0].clone(), s["v"][0].clone()
    seqs = s["seqs"].tolist()
    for i, q in enumerate(seqs):
        for r in range(cu[i], cu[i + 1]):
            at = lens[q] - cu[i + 1] + r
            k_pool[table[q][at // pg], :, at % pg] = s["k_rows"][r].view(kv, d)
            v_pool[table[q][at // pg], :, at % pg] = s["v_rows"][r].view(kv, d)
    outs, lses = [], []
    for i, q in enumerate(seqs):
        pages = torch.tensor(table[q][:_ceil(lens[q], pg)], device=k_pool.device)
        k, v = (x[pages].double().transpose(0, 1).reshape(kv, -1, d)[:, :lens[q]] for x in (k_pool, v_pool))
        rows = cu[i + 1] - cu[i]
        x = s["q"][cu[i]:cu[i + 1]].double().view(rows, kv, group, d).permute(1, 0, 2, 3).reshape(kv, rows * group, d)
        score = torch.bmm(x, k.transpose(1, 2).contiguous()).view(kv, rows, group, -1) / d ** 0.5
        for r in range(rows):
            score[:, r, :, lens[q] - rows + r + 1:] = float("-inf")
        lse = torch.logsumexp(score, 3, keepdim=True)
        o = torch.bmm(torch.exp(score - lse).reshape(kv, rows * group, -1), v.contiguous())
        outs.append(o.view(kv, rows, group, d).permute(1, 0, 2, 3).reshape(rows, heads * d))
        lses.append(lse[..., 0].permute(1, 0, 2).reshape(rows, heads))
    return {"out": torch.cat(outs), "lse": torch.cat(lses), "k": k_pool[None].double(), "v": v_pool[None].double()}


class _Book:
    """Page tables as lists, and for every place of the pool the place that its values were at in the beginning."""

    def __init__(self, s):
        self.pg = s["case"]["page"]
        self.lens = s["lens"].tolist()
        self.tables = [[p for p in row if p >= 0] for row in s["table"].tolist()]
        self.width, self.refs = s["table"].shape[1], s["refs"].tolist()
        self.origin = np.arange(len(self.refs) * self.pg).reshape(-1, self.pg)

    def fork(self, dst, src):
        old = [(list(self.tables[q]), self.lens[q]) if q >= 0 else ([], 0) for q in src]
        for q, (t, n) in zip(dst, old):
            for p in self.tables[q]:
                self.refs[p] -= 1
            for p in t:
                self.refs[p] += 1
            self.tables[q], self.lens[q] = t, n

    def reserve(self, seqs, tokens):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        free.reverse()
        holders = {}
        for q, add in zip(seqs, tokens):
            if add and self.lens[q] % self.pg:
                holders.setdefault(self.tables[q][-1], []).append(q)
        before = list(self.refs)
        for q, add in zip(seqs, tokens):
            fill = self.lens[q] % self.pg
            if add and fill:
                p = self.tables[q][-1]
                if before[p] > 1 and not (len(holders[p]) == before[p] and holders[p][0] == q):
                    to = free.pop()
                    self.origin[to, :fill] = self.origin[p, :fill]
                    self.refs[p] -= 1
                    self.refs[to] = 1
                    self.tables[q][-1] = to
            self.lens[q] += add
            while len(self.tables[q]) * self.pg < self.lens[q]:
                self.tables[q].append(free.pop())
                self.refs[self.tables[q][-1]] = 1

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        gaps = [p for p in range(n) if not self.refs[p]]
        to = dict(zip((p for p in range(n, len(self.refs)) if self.refs[p]), gaps))
        for p, h in to.items():
            self.origin[h] = self.origin[p]
            self.refs[h], self.refs[p] = self.refs[p], 0
        self.tables = [[to.get(p, p) for p in t] for t in self.tables]

    def result(self, s):
        dev, at = s["k"].device, torch.tensor(self.origin, device=s["k"].device)
        rows = [t + [-1] * (self.width - len(t)) for t in self.tables]
        pools = {x: s[x][:, at // self.pg, :, at % self.pg].permute(2, 0, 3, 1, 4).contiguous().double() for x in "kv"}
        return {"table": _ints(rows, dev), "lens": _ints(self.lens, dev), "refs": _ints(self.refs, dev), **pools}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "i8":
        x = s["x"].double()
        step = (x.abs().amax(1) / 127).float().double()  # the scale is a number of 32 bits
        whole = (x / torch.where(step > 0, step, 1.0)[:, None]).round().clamp(-127, 127)
        y = torch.matmul(whole * step[:, None], (s["w"].double() * s["w_scales"].double()[:, None]).t())
        return y if s["bias"] is None else y + s["bias"].double()
    if case["kind"] == "attn":
        return _exact_attn(s)
    book = _Book(s)
    if case["kind"] == "fork":
        book.fork(s["dst"].tolist(), s["src"].tolist())
        book.reserve(s["dst"].tolist(), s["tokens"].tolist())
    else:
        for seqs, tokens in s["sets"]:
            book.fork(seqs.tolist(), [-1] * len(seqs))
            book.compact()
            book.reserve(seqs.tolist(), tokens.tolist())
    return book.result(s)
