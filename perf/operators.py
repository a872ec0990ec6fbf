"""Cases that time and check the operators of a decode cache that is kept small: K/V held in
4 bits, the attention that reads it, attention that also accumulates each token's weight, and
eviction by that weight.

Each case is a dict; ``op`` names the operator.  ``run`` makes one pass, in plain torch or
(``own``) through ``attention_b200``.  Layout of a 4-bit pool ``(codes, scales)``: a row is
the D values of one token of one kv head in G = D / 32 groups; group j has a scale and a zero,
``scales[..., 0, j]`` and ``scales[..., 1, j]`` (fp16), and value d = 32j + 4g + i reads back as
``scale * n + zero`` with n the nibble i (low bits first) of the little-endian 16-bit word g*G + j.
"""

import math

import torch

own = False

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step's new token of a served batch: latency
        dict(name="append step", op="append", dtype="bf16", batch=4, kv_heads=8, dim=128, page=256, tokens=1, ragged=False),
        # a batch of prompts of different lengths written after prefill
        dict(name="append prompts", op="append", dtype="bf16", batch=4, kv_heads=8, dim=128, page=128, tokens=8192, ragged=True),
        # the start of a conversation: one sequence, a few pages
        dict(name="decode 512", op="decode", dtype="fp16", batch=1, q_heads=8, kv_heads=8, dim=64, page=128, context=512, ragged=False),
        # the dense decode of a long batch, every page of every sequence
        dict(name="decode 32k", op="decode", dtype="bf16", batch=8, q_heads=32, kv_heads=8, dim=128, page=128, context=32768, ragged=False),
        # a batch of unlike sequences, an odd page size and group, 32-bit queries
        dict(name="decode ragged", op="decode", dtype="fp32", batch=13, q_heads=20, kv_heads=4, dim=128, page=48, context=9001, ragged=True),
        # sparse decode at 128k: the router's pages and the local window
        dict(name="gather 128k", op="gather", dtype="bf16", batch=4, q_heads=32, kv_heads=8, dim=128, page=256, context=131072, ragged=False, window=256, top=8),
        # the dense decode of a 16-bit cache that is about to be evicted from
        dict(name="weights bf16 16k", op="weights", cache="bf16", dtype="bf16", batch=8, q_heads=32, kv_heads=8, dim=128, page=128, context=16384, ragged=False),
        # the same of a 4-bit cache with sequences of different lengths
        dict(name="weights int4 ragged", op="weights", cache="int4", dtype="fp16", batch=6, q_heads=8, kv_heads=8, dim=64, page=64, context=5000, ragged=True),
        # a long batch cut to a quarter
        dict(name="select 32k", op="select", batch=8, kv_heads=8, context=32768, budget=8192, recent=1024, ragged=False),
        # short sequences, some of them within the budget already
        dict(name="select ragged", op="select", batch=5, kv_heads=4, context=1900, budget=777, recent=100, ragged=True),
        # the move that goes with the first selection
        dict(name="compact 32k", op="compact", dtype="bf16", batch=8, kv_heads=8, dim=128, page=128, context=32768, budget=8192, recent=1024, ragged=False),
        # one sequence of a small decoder
        dict(name="compact one", op="compact", dtype="fp16", batch=1, kv_heads=8, dim=64, page=128, context=4100, budget=2048, recent=128, ragged=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["append", "decode", "gather", "weights", "select", "compact"])
    kv = _log(rng, 1, 16)
    dim = rng.choice([32, 64, 64, 96, 128, 128, 128, 256])
    batch = _log(rng, 1, 32)
    page = rng.choice([16, 32, 64, 128, 256, _log(rng, 8, 256)])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    ragged = rng.random() < 0.5
    rows = (8 << 18) * 128 // dim  # (sequence, kv head, token) rows of the largest listed cache

    def fit(most, heads):  # a length that keeps the case within the largest listed one
        return _log(rng, 1, max(1, min(most, rows // 2 // (batch * heads))))

    if op == "append":
        return dict(op=op, dtype=dtype, batch=batch, kv_heads=kv, dim=dim, page=page, tokens=fit(16384, 2 * kv),
                    ragged=ragged)
    group = rng.choice([1, 1, 2, 4, 4, 7, 8, 12])
    heads = dict(q_heads=kv * group, kv_heads=kv)
    if op == "decode":
        return dict(op=op, dtype=dtype, batch=batch, **heads, dim=dim, page=page,
                    context=fit(65536, max(kv, kv * group // 4)), ragged=ragged)
    if op == "gather":
        context = max(4 * page, fit(131072, max(kv, kv * group // 4)))
        return dict(op=op, dtype=dtype, batch=min(batch, 8), **heads, dim=dim, page=page, context=context,
                    ragged=ragged, window=rng.choice([0, page, 256, _log(rng, 1, 1000)]), top=rng.randint(1, 16))
    if op == "weights":
        return dict(op=op, cache=rng.choice(["int4", dtype]), dtype=dtype, batch=batch, **heads, dim=dim, page=page,
                    context=fit(32768, 4 * max(kv, kv * group // 4)), ragged=ragged)
    context = max(64, fit(131072 if op == "select" else 32768, kv if op == "select" else 4 * kv))
    budget = round(context * rng.uniform(0.1, 0.9))
    recent = rng.choice([0, round(budget * rng.uniform(0, 0.5))])
    some = dict(batch=batch, kv_heads=kv, context=context, budget=budget, recent=recent, ragged=ragged)
    return dict(op=op, **some) if op == "select" else dict(op=op, dtype=dtype, dim=dim, page=page, **some)


# ------------------------------------------------------------------------------ inputs
def _lens(c, most, g):
    """Lengths of the batch: all ``most``, or anything up to it with the longest kept."""
    n = torch.full((c["batch"],), most, dtype=torch.int32, device="cuda")
    if c["ragged"]:
        n = (torch.rand(c["batch"], generator=g, device="cuda") * most).to(torch.int32) + 1
        n[0] = most
    return n


def _paging(c, most, g):
    """A seeded scatter of the sequences' pages through the pool."""
    pages = -(-most // c["page"])
    n = c["batch"] * pages
    return n, torch.randperm(n, generator=g, device="cuda").to(torch.int32).view(c["batch"], pages)


def _states(shape, g):
    """Keys or values as a model makes them: unit-scale channels, some of them stronger."""
    x = torch.randn(shape, generator=g, device="cuda")
    return x * (0.5 + torch.rand(shape[-1], generator=g, device="cuda") ** 4 * 3)


def _weights(shape, g):
    """Accumulated attention: heavy-tailed, with tokens that nothing ever looked at (ties)."""
    w = torch.exp(2 * torch.randn(shape, generator=g, device="cuda") - 4)
    return w * (torch.rand(shape, generator=g, device="cuda") > 0.05)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=c)
    if c["op"] == "append":
        t = c["tokens"]
        s["positions"] = torch.randint(0, 2 * c["page"], (c["batch"],), generator=g, device="cuda").to(torch.int32)
        n, s["table"] = _paging(c, t + 2 * c["page"], g)
        shape = (c["batch"], c["kv_heads"], t, c["dim"])
        s["k_new"], s["v_new"] = (_states(shape, g).to(DT[c["dtype"]]) for _ in range(2))
        s["new_lens"] = _lens(c, t, g)
        s["k"], s["v"] = (_empty_int4(n, c) for _ in range(2))
        return s
    s["lens"] = _lens(c, c["context"], g)
    if c["op"] in ("select", "compact"):
        s["weights"] = _weights((c["batch"], c["kv_heads"], c["context"]), g)
    if c["op"] == "select":
        return s
    n, s["table"] = _paging(c, c["context"], g)
    shape = (n, c["kv_heads"], c["page"], c["dim"])
    if c["op"] == "compact":
        s["keep"], s["kept"] = _select(s["weights"], s["lens"], c["budget"], c["recent"])
        s["k"], s["v"] = (_states(shape, g).to(DT[c["dtype"]]) for _ in range(2))
        return s
    s["q"] = torch.randn(c["batch"], c["q_heads"], c["dim"], generator=g, device="cuda").to(DT[c["dtype"]])
    kind = c.get("cache", "int4")
    s["k"], s["v"] = (_quantise(_states(shape, g)) if kind == "int4" else _states(shape, g).to(DT[kind])
                      for _ in range(2))
    if c["op"] == "gather":
        # the router picks among the pages older than the window; slots it cannot fill hold -1
        old = ((s["lens"] - c["window"]).clamp(min=0) // c["page"])[:, None]
        score = torch.rand(c["batch"], max(s["table"].size(1), c["top"]), generator=g, device="cuda")
        page = torch.arange(score.size(1), device="cuda")
        score = torch.where(page < old, score, -1.0)
        top = score.topk(c["top"], 1)
        s["selected"] = torch.where(top.values >= 0, top.indices, -1)
    if c["op"] == "weights":
        # what some tens of earlier steps left there
        s["weights"] = torch.rand(c["batch"], c["kv_heads"], c["context"], generator=g, device="cuda")
        s["weights"] *= 64 * c["q_heads"] / c["kv_heads"] / c["context"]
    return s


def _empty_int4(pages, c):
    rows = (pages, c["kv_heads"], c["page"])
    return (torch.zeros(*rows, c["dim"] // 2, dtype=torch.uint8, device="cuda"),
            torch.zeros(*rows, 2, c["dim"] // 32, dtype=torch.float16, device="cuda"))


# ------------------------------------------------------------------------------ plain forms
def _quantise(x):
    """Codes and scales of fp32 values, by the operator's own steps in fp32."""
    x = x.float().unflatten(-1, (-1, 32))
    low, high = x.amin(-1), x.amax(-1)
    scale = ((high - low) / 15).clamp(max=65504).half()
    zero = low.clamp(-65504, 65504).half()
    n = ((x - zero.float()[..., None]) / scale.float()[..., None]).round().clamp(0, 15)
    n = torch.where(scale[..., None] > 0, n, 0)
    bad = ~x.isfinite().all(-1)
    n = torch.where(bad[..., None], 0, n).to(torch.uint8)
    scale, zero = (torch.where(bad, torch.nan, t).half() for t in (scale, zero))
    n = n.unflatten(-1, (8, 2, 2)).transpose(-4, -3).contiguous()  # [..., 8 words, G, 2 bytes, 2 nibbles]
    return (n[..., 0] | (n[..., 1] << 4)).flatten(-3), torch.stack((scale, zero), -2)


def _values(pool):
    """The fp32 values a 4-bit pool stands for."""
    codes, scales = pool
    b = codes.unflatten(-1, (8, -1, 2))
    n = torch.stack((b & 15, b >> 4), -1).transpose(-4, -3).flatten(-3).float()
    scale, zero = scales.float().unbind(-2)
    return (n * scale[..., None] + zero[..., None]).flatten(-2)


def _in_order(pool, table):
    """[pages, Hkv, P, ...] through the table: [B, Hkv, tokens, ...]."""
    return pool[table.long()].transpose(1, 2).flatten(2, 3)


def _attend(q, k, v, valid):
    """softmax(q k^T / sqrt(D)) and its product with v over the valid tokens [B, N], in fp32."""
    q = q.float().unflatten(1, (k.size(1), -1))
    score = (q @ k.transpose(2, 3)) / math.sqrt(k.size(3))
    score = torch.where(valid[:, None, None], score, -torch.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return (p @ v).flatten(1, 2), p.sum(2)


def _select(w, lens, budget, recent):
    idx = torch.arange(w.size(2), device=w.device)
    lens = lens.long()[:, None, None]
    key = torch.where(idx >= lens - min(recent, budget), torch.inf, w)
    key = torch.where(idx >= lens, -1.0, key)  # weights are sums of probabilities: never negative
    order = torch.sort(key, dim=2, descending=True, stable=True).indices[:, :, :budget]
    none = torch.iinfo(torch.int64).max
    keep = torch.where(order < lens, order, none).sort(2).values
    return torch.where(keep == none, -1, keep).to(torch.int32), lens.flatten().clamp(max=budget).to(torch.int32)


def _compact(pool, table, keep):
    page = pool.size(2)
    b = torch.arange(keep.size(0), device=keep.device)[:, None, None]
    h = torch.arange(keep.size(1), device=keep.device)[None, :, None]
    to = torch.arange(keep.size(2), device=keep.device)
    src = torch.where(keep >= 0, keep.long(), to)
    table = table.long()
    pool[table[b, to // page], h, to % page] = pool[table[b, src // page], h, src % page]


def run(state):
    c, s = state["case"], state
    if own:
        import attention_b200 as spa
    if c["op"] == "append":
        if own:
            spa.kv_append_int4(s["k"], s["v"], s["table"], s["k_new"], s["v_new"], s["positions"],
                               new_lens=s["new_lens"])
            return spa.kv_read_int4(s["k"], s["v"], s["table"], s["positions"], c["tokens"], lens=s["new_lens"],
                                    dtype=DT[c["dtype"]])
        there = torch.arange(c["tokens"], device="cuda") < s["new_lens"][:, None]
        return tuple(torch.where(there[:, None, :, None], _values(_quantise(x)), 0).to(x.dtype)
                     for x in (s["k_new"], s["v_new"]))
    if c["op"] == "select":
        if own:
            return spa.select_tokens(s["weights"], s["lens"], budget=c["budget"], recent=c["recent"])
        return _select(s["weights"], s["lens"], c["budget"], c["recent"])
    if c["op"] == "compact":
        if own:
            spa.compact_tokens((s["k"], s["v"]), s["table"], s["keep"], weights=s["weights"])
        else:
            _compact(s["k"], s["table"], s["keep"])
            _compact(s["v"], s["table"], s["keep"])
            w = s["weights"].gather(2, s["keep"].long().clamp(min=0))
            s["weights"].zero_()
            s["weights"][:, :, : c["budget"]] = torch.where(s["keep"] >= 0, w, 0)
        return s["k"], s["v"], s["weights"]
    if own:
        more = dict(page_table=s["table"], context_lens=s["lens"])
        if c["op"] == "gather":
            return spa.paged_gather_decode_attention_int4(s["q"], s["k"], s["v"], s["selected"],
                                                          local_window=c["window"], block_size=c["page"], **more)
        if c["op"] == "weights":
            f = spa.paged_decode_attention_int4 if c["cache"] == "int4" else spa.paged_decode_attention
            return f(s["q"], s["k"], s["v"], weights=s["weights"], **more), s["weights"]
        return spa.paged_decode_attention_int4(s["q"], s["k"], s["v"], **more)
    lens = s["lens"].long()[:, None]
    if c["op"] == "gather":
        w, page = c["window"], c["page"]
        local = lens - w + torch.arange(w, device="cuda")
        far = (s["selected"][..., None] * page + torch.arange(page, device="cuda")).flatten(1)
        token = torch.cat((local, torch.where((s["selected"] >= 0).repeat_interleave(page, 1), far, -1)), 1)
        valid = (token >= 0) & (token < lens)
        token = torch.where(valid, token, 0)
        at = s["table"].long().gather(1, token // page)
        k, v = (_values(tuple(t[at, :, token % page] for t in s[x])).transpose(1, 2) for x in ("k", "v"))
        return _attend(s["q"], k, v, valid)[0].to(s["q"].dtype)
    if c.get("cache", "int4") == "int4":
        k, v = (_values(tuple(_in_order(t, s["table"]) for t in s[x])) for x in ("k", "v"))
    else:
        k, v = (_in_order(s[x], s["table"]).float() for x in ("k", "v"))
    out, p = _attend(s["q"], k, v, torch.arange(k.size(2), device="cuda") < lens)
    out = out.to(s["q"].dtype)
    if c["op"] == "weights":
        s["weights"] += p[:, :, : c["context"]]
        return out, s["weights"]
    return out


# ------------------------------------------------------------------------------ work
def work(case):
    """Bytes and operations of the full-length case (ragged ones: the mean length of _lens)."""
    c = case
    share = (1 + (c["batch"] - 1) / 2) / c["batch"] if c["ragged"] else 1.0
    heads = c["batch"] * c["kv_heads"]
    if c["op"] == "select":
        n = heads * c["context"] * share
        return {"bytes": 4 * n + 4 * heads * c["budget"], "flops": n}
    es = 4 if c.get("dtype") == "fp32" else 2
    if c["op"] == "append":
        n = heads * c["tokens"] * share * c["dim"]
        full = heads * c["tokens"] * c["dim"]  # the read-back returns padded rows as zeros
        return {"bytes": 2 * (n * (es + 2 * 0.625) + full * es), "flops": 2 * 8 * n}
    if c["op"] == "compact":
        kept = sum(min(c["budget"], n) for n in ([c["context"]] + [c["context"] / 2 if c["ragged"] else c["context"]]
                                                 * (c["batch"] - 1))) * c["kv_heads"]
        return {"bytes": 2 * 2 * kept * c["dim"] * es + 8 * kept + 4 * heads * c["context"], "flops": 0}
    n = heads * c["context"] * share
    if c["op"] == "gather":
        n = heads * min(c["context"] * share, c["window"] + c["top"] * c["page"])
    row = c["dim"] * 0.625 if c.get("cache", "int4") == "int4" else c["dim"] * (4 if c["cache"] == "fp32" else 2)
    q = c["batch"] * c["q_heads"] * c["dim"]
    more = 8 * n if c["op"] == "weights" else 0
    return {"bytes": 2 * n * row + 2 * q * es + more, "flops": 4 * n * c["dim"] * c["q_heads"] / c["kv_heads"]}


# ------------------------------------------------------------------------------ 64-bit results
def _values64(pool):
    codes, scales = pool
    groups = scales.size(-1)
    d = torch.arange(32 * groups, device=codes.device)
    word = (d % 32 // 4) * groups + d // 32
    n = codes[..., 2 * word + d % 4 // 2] >> (4 * (d % 2)).to(torch.uint8) & 15
    scales = scales.double()[..., d // 32]
    return scales[..., 0, :] * n.double() + scales[..., 1, :]


def _rows64(pool, table, token):
    """Rows [Hkv, N, D] of one sequence's tokens in 64 bits."""
    rows = lambda t: t[table[token // t.size(2)].long(), :, token % t.size(2)]  # noqa: E731
    return (_values64(tuple(rows(t) for t in pool)) if isinstance(pool, tuple) else rows(pool).double()).transpose(0, 1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "append":
        # the rounding of scales, zeros and codes belongs to the definition: fp32 steps, as numpy takes them
        import numpy as np

        outs = []
        for x in (s["k_new"], s["v_new"]):
            out = torch.zeros(x.shape, dtype=torch.float64)
            for b, n in enumerate(s["new_lens"].tolist()):
                a = x[b, :, :n].float().cpu().numpy().reshape(x.size(1), n, -1, 32)
                low, high = a.min(-1, keepdims=True), a.max(-1, keepdims=True)
                scale = ((high - low) / np.float32(15)).astype(np.float16).astype(np.float32)
                zero = low.astype(np.float16).astype(np.float32)
                with np.errstate(divide="ignore", invalid="ignore"):
                    code = np.clip(np.rint((a - zero) / scale), 0, 15)
                code = np.where(scale > 0, code, 0).astype(np.float64)
                out[b, :, :n] = torch.from_numpy(scale.astype(np.float64) * code + zero).flatten(-2)
            outs.append(out)
        return tuple(outs)
    if c["op"] == "select":
        w, keep = s["weights"].double().cpu(), torch.full((c["batch"], c["kv_heads"], c["budget"]), -1)
        lens = s["lens"].tolist()
        for b, n in enumerate(lens):
            recent = min(c["recent"], c["budget"])
            for h in range(c["kv_heads"]):
                chosen = range(n)
                if n > c["budget"]:
                    value, _ = w[b, h, : n - recent].sort(descending=True)
                    more = c["budget"] - recent
                    if more:
                        old = w[b, h, : n - recent]
                        above = (old > value[more - 1]).nonzero().flatten()
                        equal = (old == value[more - 1]).nonzero().flatten()[: more - above.numel()]
                        chosen = sorted(above.tolist() + equal.tolist()) + list(range(n - recent, n))
                    else:
                        chosen = range(n - recent, n)
                keep[b, h, : len(chosen)] = torch.tensor(list(chosen))
        return keep, torch.tensor([min(n, c["budget"]) for n in lens])
    if c["op"] == "compact":
        k, v, w = s["k"].double(), s["v"].double(), torch.zeros_like(s["weights"], dtype=torch.float64)
        for b in range(c["batch"]):
            n = int(s["kept"][b])
            to = torch.arange(n, device="cuda")
            page = s["table"][b].long()
            for h in range(c["kv_heads"]):
                src = s["keep"][b, h, :n].long()
                for new, old in ((k, s["k"]), (v, s["v"])):
                    new[page[to // c["page"]], h, to % c["page"]] = old[page[src // c["page"]], h, src % c["page"]].double()
                w[b, h, :n] = s["weights"][b, h, src].double()
        return k, v, w
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    acc = s["weights"].double() if c["op"] == "weights" else None
    for b, n in enumerate(s["lens"].tolist()):
        token = torch.arange(n, device="cuda")
        if c["op"] == "gather":
            token = [token[max(0, n - c["window"]):]]
            token += [torch.arange(p * c["page"], min((p + 1) * c["page"], n), device="cuda")
                      for p in s["selected"][b].tolist() if p >= 0]
            token = torch.cat(token)
        if not token.numel():
            continue
        k, v = (_rows64(s[x], s["table"][b], token) for x in ("k", "v"))
        q = s["q"][b].double().view(c["kv_heads"], -1, c["dim"])
        p = torch.softmax(torch.einsum("hgd,hnd->hgn", q, k) / c["dim"] ** 0.5, -1)
        out[b] = torch.einsum("hgn,hnd->hgd", p, v).flatten(0, 1)
        if acc is not None:
            acc[b, :, :n] += p.sum(1)
    return (out, acc) if acc is not None else out
