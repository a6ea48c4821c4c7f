"""Cases of the serving operators over an INT8 KV cache and over logits: quantised append and read-back, attention
of one or several tokens per sequence (chains, drafted trees, prompt chunks), and token picks under rules.

`run` computes an operator in plain torch, or, where `own` is set, through the package's entry points."""
import math

import torch

own = False

DEV = "cuda"
VOCAB = 151936  # the vocabulary of the published decoders


# ------------------------------------------------------------------ cases --
def listed():
    gqa = dict(n_kv=8, group=2, hd=128)  # both published decoders: 16 query heads over 8 kv heads of 128
    return [
        # one decode step of a full batch: one new row per sequence, quantised and read back
        dict(name="append_step_m8", op="append", seqs=8, rows=1, past=1000, n_kv=8, hd=128, gather=False),
        # the prompts of a batch of 30 s segments (about 404 rows each), written once and read back for the prefill
        dict(name="append_prompt_m8", op="append", seqs=8, rows=404, past=0, n_kv=8, hd=128, gather=False),
        # the accepted nodes of drafted trees, gathered from the rows of all nodes, on top of long histories
        dict(name="append_accepted_m61", op="append", seqs=61, rows=17, past=1500, n_kv=8, hd=128, gather=True),
        # one segment's whole history handed to an f32 consumer
        dict(name="read_m1", op="read", seqs=1, rows=551, past=0, n_kv=8, hd=128),
        # the histories of many streams
        dict(name="read_m16", op="read", seqs=16, rows=2040, past=8, n_kv=8, hd=128),
        # one stream decoding a 30 s segment: latency
        dict(name="decode_m1", op="attend", seqs=1, rows=1, past=544, tree=False, ragged=False, **gqa),
        # many streams with long, ragged histories: cache bandwidth
        dict(name="decode_m32_long", op="attend", seqs=32, rows=1, past=8000, tree=False, ragged=True, **gqa),
        # a small model without shared heads, head_dim 64, an odd batch
        dict(name="decode_m5_hd64", op="attend", seqs=5, rows=1, past=1777, tree=False, ragged=True, n_kv=6, group=1,
             hd=64),
        # verification of drafted trees for a batch of streams
        dict(name="tree_m8", op="attend", seqs=8, rows=31, past=1100, tree=True, ragged=True, **gqa),
        # prompt chunks of 30 s segments over the quantised cache
        dict(name="prompt_m4", op="attend", seqs=4, rows=404, past=0, tree=False, ragged=True, **gqa),
        # the pick of one stream under a repetition penalty: latency
        dict(name="pick_m1", op="pick", rows=1, vocab=VOCAB, history=120, bias=0, mask=False),
        # the picks of all nodes of a batch of drafted trees, every rule on
        dict(name="pick_m64", op="pick", rows=64, vocab=VOCAB, history=400, bias=24, mask=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    cap = max(work(c)["bytes"] for c in listed())
    most = max(work(c)["flops"] for c in listed())
    while True:
        op = rng.choice(["append", "read", "attend", "attend", "pick"])
        n_kv, hd = rng.randint(1, 8), rng.choice([64, 128])
        if op == "append":
            c = dict(op=op, seqs=_log(rng, 1, 64), rows=_log(rng, 1, 500), past=rng.randint(0, 2000), n_kv=n_kv, hd=hd,
                     gather=rng.random() < 0.4)
        elif op == "read":
            c = dict(op=op, seqs=_log(rng, 1, 24), rows=_log(rng, 1, 2048), past=rng.randint(0, 300), n_kv=n_kv, hd=hd)
        elif op == "attend":
            kind = rng.choice(["decode", "tree", "chunk"])
            rows = 1 if kind == "decode" else rng.randint(2, 64) if kind == "tree" else _log(rng, 2, 500)
            c = dict(op=op, seqs=_log(rng, 1, 40), rows=rows, past=_log(rng, 1, 9000), tree=kind == "tree",
                     ragged=rng.random() < 0.7, n_kv=n_kv, group=rng.choice([1, 2, 3, 4, 7, 8]), hd=hd)
        else:
            c = dict(op=op, rows=_log(rng, 1, 64), vocab=rng.choice([VOCAB, _log(rng, 1000, VOCAB)]),
                     history=_log(rng, 1, 1500), bias=rng.randint(0, 64), mask=rng.random() < 0.6)
        w = work(c)
        if w["bytes"] <= cap and w["flops"] <= most:
            return c


# ------------------------------------------------------------------- sizes --
def _lengths(case):
    """(past, rows) of each sequence: a fixed spread of the case's sizes, no randomness."""
    n = case["seqs"]
    past, rows = [case["past"]] * n, [case["rows"]] * n
    if case["op"] == "append" and case["gather"]:
        rows = [1 + (case["rows"] - 1) * (i % 5) // 4 for i in range(n)]  # accepted nodes differ by sequence
    if case.get("ragged"):
        past = [case["past"] * (n - i) // n for i in range(n)]
        if case["rows"] > 1:
            rows = [max(1, case["rows"] - (case["rows"] // 3) * (i % 3) // 2) for i in range(n)]
    return past, rows


def work(case):
    if case["op"] == "pick":
        m, v = case["rows"], case["vocab"]
        b = m * (8 * v + 4 + 4 * case["history"] + 8 * case["bias"] + (v / 8 if case["mask"] else 0))
        return {"bytes": int(b), "flops": m * v}
    past, rows = _lengths(case)
    d, h = case["n_kv"] * case["hd"], case["n_kv"]
    codes = 2 * d + 8 * h  # K and V codes and scales of a cache row
    if case["op"] == "append":  # f32 rows in, codes out, f32 rows back
        return {"bytes": sum(rows) * (8 * d + codes + 8 * d), "flops": sum(rows) * 6 * d}
    if case["op"] == "read":
        return {"bytes": sum(rows) * (codes + 8 * d), "flops": sum(rows) * 2 * d}
    heads = case["n_kv"] * case["group"]
    seen = sum(r * p + r * (r + 1) // 2 for p, r in zip(past, rows))  # pairs of a query and a key it may see
    b = sum(p + r for p, r in zip(past, rows)) * codes + sum(rows) * 8 * heads * case["hd"]
    return {"bytes": b, "flops": 4 * heads * case["hd"] * seen}


# ----------------------------------------------------------------- prepare --
def _starts(counts):
    t = torch.zeros(len(counts) + 1, dtype=torch.int32)
    t[1:] = torch.tensor(counts).cumsum(0)
    return t.to(DEV)


def _codes(x, hd):
    """Rows quantised head by head: int8 codes and f32 scales."""
    h = x.view(*x.shape[:-1], -1, hd)
    top = h.abs().amax(-1)
    most = torch.full_like(top, 127.0)  # a tensor: dividing by or into a Python number is a product with a reciprocal
    inv = torch.where(top > 0, most / top, torch.zeros_like(top))
    a = (h * inv[..., None]).abs()
    low = a.floor()
    c = (low + (a - low >= 0.5)).copysign(h).clamp(-128, 127)
    return c.to(torch.int8).view(x.shape), top / most


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if case["op"] == "pick":
        return _prepare_pick(case, seed, g)
    past, rows = _lengths(case)
    n, n_kv, hd, layers, layer = case["seqs"], case["n_kv"], case["hd"], 2, 1
    total, longest = sum(rows), max(p + r for p, r in zip(past, rows))
    max_seq, d = longest + 9, n_kv * hd
    cpu = torch.Generator().manual_seed(seed + 1)
    st = {
        "case": case, "layer": layer, "longest": longest, "most_rows": max(rows), "total": total,
        "k": torch.zeros(n, layers, max_seq, d, dtype=torch.int8, device=DEV),
        "v": torch.zeros(n, layers, max_seq, d, dtype=torch.int8, device=DEV),
        "ks": torch.zeros(n, layers, max_seq, n_kv, device=DEV),
        "vs": torch.zeros(n, layers, max_seq, n_kv, device=DEV),
        "starts": _starts(rows), "positions": torch.tensor(past, dtype=torch.int32).to(DEV),
        "slots": torch.randperm(n, generator=cpu).to(torch.int32).to(DEV),  # sequences sit in any slot
    }
    if case["op"] == "append":
        n_src = total * 2 if case["gather"] else total
        st["k_new"], st["v_new"] = randn(n_src, d), randn(n_src, d)
        st["src"] = None
        if case["gather"]:
            st["src"] = torch.randperm(n_src, generator=cpu)[:total].to(torch.int32).to(DEV)
    else:
        for i in range(n):  # a history as a decoder leaves it: normal rows, head by head of their own size
            for code, scale in (("k", "ks"), ("v", "vs")):
                size = torch.rand(1, n_kv, 1, generator=g, device=DEV) + 0.5
                x = (randn(longest, n_kv, hd) * size).view(longest, d)
                st[code][i, layer, :longest], st[scale][i, layer, :longest] = _codes(x, hd)
    if case["op"] == "attend":
        heads = n_kv * case["group"]
        st["q"] = randn(total, heads * hd)
        st["out"] = torch.empty_like(st["q"])
        st["scale"] = 1.0 / math.sqrt(hd)
        st["mask"] = _tree_masks(rows, cpu) if case["tree"] else None
    else:
        st["k_out"], st["v_out"] = torch.empty(total, d, device=DEV), torch.empty(total, d, device=DEV)
    if own:
        from qwenasr_b200.kvcache import KvCacheInt8, KvRows
        st["cache"] = KvCacheInt8(st["k"], st["v"], st["ks"], st["vs"])
        st["rows"] = KvRows(st["starts"], st["positions"], st["slots"], n_rows=total, max_rows=st["most_rows"])
    return st


def _tree_masks(rows, cpu):
    """Ancestor masks of random drafted trees: node t hangs below any earlier node, row 0 is the root."""
    masks = []
    for r in rows:
        up = [0] * r
        for t in range(r):
            parent = -1 if t == 0 else int(torch.randint(max(0, t - 6), t, (1,), generator=cpu))
            up[t] = (up[parent] if t else 0) | (1 << t)
        masks += [u - (1 << 64) if u >> 63 else u for u in up]
    return torch.tensor(masks, dtype=torch.int64).to(DEV)


def _prepare_pick(case, seed, g):
    m, v = case["rows"], case["vocab"]
    cpu = torch.Generator().manual_seed(seed + 1)
    logits = torch.randn(m, v, generator=g, device=DEV) * 2.5
    st = {"case": case, "logits": logits, "out": torch.empty_like(logits),
          "ids": torch.empty(m, dtype=torch.int32, device=DEV)}
    h = case["history"]
    counts = [1 + (h - 1) * (m - i) // m for i in range(m)]
    # transcripts repeat: tokens come from a small set, among them the likeliest ones
    pool = torch.cat([logits.topk(min(8, v), dim=1).indices.cpu(),
                      torch.randint(0, v, (m, max(1, h // 2)), generator=cpu)], dim=1)
    hist = [pool[i][torch.randint(0, pool.shape[1], (c,), generator=cpu)] for i, c in enumerate(counts)]
    st["hist"], st["hist_starts"] = torch.cat(hist).to(torch.int32).to(DEV), _starts(counts)
    st["rep"] = (1.0 + torch.rand(m, generator=cpu) * 0.5).to(DEV)
    st["pres"], st["freq"] = (torch.rand(m, generator=cpu) * 0.6).to(DEV), (torch.rand(m, generator=cpu) * 0.2).to(DEV)
    st["bias_ids"] = st["bias_vals"] = st["bias_starts"] = st["mask"] = None
    if case["bias"]:
        n = [max(1, case["bias"] * (i % 4 + 1) // 4) for i in range(m)]
        ids = [torch.randperm(v, generator=cpu)[:c] for c in n]
        st["bias_ids"], st["bias_starts"] = torch.cat(ids).to(torch.int32).to(DEV), _starts(n)
        st["bias_vals"] = (torch.randn(sum(n), generator=cpu) * 3).to(DEV)
    if case["mask"]:
        # a grammar allows anything from a handful of tokens to most of them
        words = (v + 31) // 32
        share = torch.rand(m, 1, generator=g, device=DEV) ** 3
        bits = (torch.rand(m, words * 32, generator=g, device=DEV) < share).view(m, words, 32).to(torch.int64)
        w = (bits << torch.arange(32, device=DEV)).sum(-1)
        st["mask"] = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)
    return st


# --------------------------------------------------------------------- run --
def run(state):
    op = state["case"]["op"]
    if own:
        return _own(op, state)
    if op == "append":
        return _plain_append(state)
    if op == "read":
        return _plain_read(state)
    return _plain_attend(state) if op == "attend" else _plain_pick(state)


def _own(op, s):
    from qwenasr_b200 import kernels as K
    if op == "append":
        K.kv_append_int8(s["cache"], s["layer"], s["rows"], s["k_new"], s["v_new"], s["src"])
        K.kv_read_int8(s["k_out"], s["v_out"], s["cache"], s["layer"], s["rows"])
        return s["k_out"], s["v_out"]
    if op == "read":
        K.kv_read_int8(s["k_out"], s["v_out"], s["cache"], s["layer"], s["rows"])
        return s["k_out"], s["v_out"]
    if op == "attend":
        heads = s["case"]["n_kv"] * s["case"]["group"]
        K.tree_attention_int8(s["out"], s["q"], s["cache"], s["layer"], s["rows"], heads, s["scale"], s["mask"])
        return s["out"]
    K.logits_pick(s["ids"], s["out"], s["logits"], s["case"]["rows"], s["case"]["vocab"], history=s["hist"],
                  history_starts=s["hist_starts"], repetition=s["rep"], presence=s["pres"], frequency=s["freq"],
                  bias_ids=s["bias_ids"], bias_values=s["bias_vals"], bias_starts=s["bias_starts"],
                  allow_mask=s["mask"])
    return s["ids"], s["out"]


def _where(s):
    """Slot and cache row of each packed row."""
    r = torch.arange(s["total"], device=DEV)
    m = (s["starts"][1:, None] <= r).sum(0)
    return s["slots"][m].long(), (s["positions"][m] + r - s["starts"][m]).long()


def _plain_append(s):
    hd, layer = s["case"]["hd"], s["layer"]
    slot, pos = _where(s)
    for new, code, scale in (("k_new", "k", "ks"), ("v_new", "v", "vs")):
        x = s[new] if s["src"] is None else s[new][s["src"].long()]
        s[code][slot, layer, pos], s[scale][slot, layer, pos] = _codes(x, hd)
    return _plain_read(s)


def _plain_read(s):
    hd, layer = s["case"]["hd"], s["layer"]
    slot, pos = _where(s)

    def back(code, scale):
        c = s[code][slot, layer, pos].float()
        return (c.view(s["total"], -1, hd) * s[scale][slot, layer, pos][..., None]).view(s["total"], -1)

    return back("k", "ks"), back("v", "vs")


def _plain_attend(s):
    c, layer, top = s["case"], s["layer"], s["longest"]
    n, n_kv, g, hd, t = c["seqs"], c["n_kv"], c["group"], c["hd"], s["most_rows"]
    slot = s["slots"].long()

    def whole(code, scale):  # [n, n_kv, keys, hd]
        x = s[code][slot, layer, :top].float().view(n, top, n_kv, hd) * s[scale][slot, layer, :top][..., None]
        return x.transpose(1, 2)

    step = torch.arange(t, device=DEV)
    count = s["starts"][1:] - s["starts"][:-1]
    row = torch.minimum(s["starts"][:-1, None] + step, s["starts"][1:, None] - 1).long()  # [n, t], short ones padded
    q = s["q"].view(s["total"], n_kv, g, hd)[row].permute(0, 2, 3, 1, 4).reshape(n, n_kv, g * t, hd)
    key = torch.arange(top, device=DEV)[None, None] - s["positions"][:, None, None]  # place in the tree, below 0: past
    if s["mask"] is None:
        seen = key <= step[None, :, None]
    else:
        inside = (s["mask"][row][..., None] >> key.clamp(0, 63)) & 1
        seen = (key < 0) | ((key < count[:, None, None]) & (inside == 1))
    score = (q @ whole("k", "ks").transpose(2, 3)).view(n, n_kv, g, t, top) * s["scale"]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    e = (score - score.amax(-1, keepdim=True)).exp()
    out = (e.view(n, n_kv, g * t, top) @ whole("v", "vs")).view(n, n_kv, g, t, hd) / e.sum(-1, keepdim=True)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, t, -1)
    r = torch.arange(s["total"], device=DEV)
    m = (s["starts"][1:, None] <= r).sum(0)
    return out[m, (r - s["starts"][m]).long()]


def _plain_pick(s):
    m, v = s["case"]["rows"], s["case"]["vocab"]
    x = s["logits"]
    r = torch.arange(s["hist"].numel(), device=DEV)
    row = (s["hist_starts"][1:, None] <= r).sum(0)
    n = torch.zeros(m, v, device=DEV)
    n.index_put_((row, s["hist"].long()), torch.ones_like(r, dtype=torch.float32), accumulate=True)
    rep = s["rep"][:, None]
    y = torch.where(x > 0, x / rep, x * rep) - (s["pres"][:, None] + s["freq"][:, None] * n)
    x = torch.where(n > 0, y, x)
    if s["bias_ids"] is not None:
        r = torch.arange(s["bias_ids"].numel(), device=DEV)
        row = (s["bias_starts"][1:, None] <= r).sum(0)
        add = torch.zeros(m, v, device=DEV)
        add[row, s["bias_ids"].long()] = s["bias_vals"]
        x = x + add
    none = torch.zeros(m, dtype=torch.bool, device=DEV)
    if s["mask"] is not None:
        may = ((s["mask"][:, :, None] >> torch.arange(32, device=DEV)) & 1).view(m, -1)[:, :v] == 1
        x = x.masked_fill(~may, -math.inf)
        none = ~may.any(-1)
    top = x.amax(-1, keepdim=True)
    place = torch.where(x == top, torch.arange(v, device=DEV), v).amin(-1)
    return torch.where(none, -1, place).to(torch.int32), x


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pick":
        return _exact_pick(case, s)
    hd, n_kv, layer = case["hd"], case["n_kv"], s["layer"]
    past, rows = _lengths(case)
    slots = s["slots"].tolist()
    if case["op"] == "append":
        outs = []
        for new in (s["k_new"], s["v_new"]):
            x = new.double() if s["src"] is None else new.double()[s["src"].long()]
            x = x.view(-1, n_kv, hd)
            top = x.abs().max(-1, keepdim=True).values
            # the rule of the quantised files: 127 / top and its product with x are f32 values (the product of two
            # f32 values is exact in 64 bits before it is rounded), halves go away from zero
            t = (x * (127 / top).float().double()).float().double()
            outs.append((torch.trunc(t + 0.5 * torch.sign(t)) * (top / 127)).view(-1, n_kv * hd))
        return tuple(outs)

    def rows_of(code, scale, i, a, b):
        x = s[code][slots[i], layer, a:b].double().view(b - a, n_kv, hd)
        return x * s[scale][slots[i], layer, a:b].double()[..., None]

    if case["op"] == "read":
        return tuple(torch.cat([rows_of(c, sc, i, p, p + r).flatten(1) for i, (p, r) in enumerate(zip(past, rows))])
                     for c, sc in (("k", "ks"), ("v", "vs")))
    out, at = [], 0
    for i, (p, r) in enumerate(zip(past, rows)):
        k, v = rows_of("k", "ks", i, 0, p + r), rows_of("v", "vs", i, 0, p + r)
        q = s["q"][at:at + r].double().view(r, n_kv, case["group"], hd)
        may = torch.ones(r, p + r, dtype=torch.bool)
        if s["mask"] is None:
            may[:, p:] = torch.tril(torch.ones(r, r, dtype=torch.bool))
        else:
            may[:, p:] = torch.tensor([[w >> j & 1 for j in range(r)] for w in s["mask"][at:at + r].tolist()]) == 1
        score = torch.einsum("rhgd,khd->rhgk", q, k) * s["scale"]
        score[~may.to(DEV)[:, None, None].expand_as(score)] = -math.inf
        out.append(torch.einsum("rhgk,khd->rhgd", score.softmax(-1), v).reshape(r, -1))
        at += r
    return torch.cat(out)


def _exact_pick(case, s):
    m, v = case["rows"], case["vocab"]
    x = s["logits"].double()
    hs = s["hist_starts"].tolist()
    bs = s["bias_starts"].tolist() if s["bias_starts"] is not None else None
    ids = []
    for i in range(m):
        tok, n = s["hist"][hs[i]:hs[i + 1]].long().unique(return_counts=True)
        l, rep = x[i, tok], s["rep"][i].double()
        x[i, tok] = torch.where(l > 0, l / rep, l * rep) - s["pres"][i].double() - s["freq"][i].double() * n
        if bs:
            x[i].index_add_(0, s["bias_ids"][bs[i]:bs[i + 1]].long(), s["bias_vals"][bs[i]:bs[i + 1]].double())
        if s["mask"] is not None:
            word = s["mask"][i].long()[:, None].bitwise_right_shift(torch.arange(32, device=DEV))
            x[i][(word & 1).flatten()[:v] == 0] = -math.inf
        ids.append(int(x[i].argmax()) if bool((x[i] > -math.inf).any()) else -1)
    return torch.tensor(ids, dtype=torch.int32), x
