"""The operators of a serving step over a paged KV cache, in a plain form and as the framework's calls.

Keys and values live in a pool of pages, [n_pages][n_kv][page][head_dim] in f32 or f16; entry j of a sequence is slot
j % page of page table[sequence][j // page]. Kinds of case:

* ``append``  — new q / k / v rows (f32, fused) rotated to their positions, the keys and values into their pages.
* ``attention``  — the query rows of one or several new tokens per sequence over their pages; the first `shared` entries of
  all sequences are the same ones (a common system prompt).
* ``sample``  — the next token of every row of logits: temperature, top-k, top-p, min-p and given uniform numbers.

Head layouts are those of the repository's configurations: 32 heads / 8 KV heads of 128, 8 / 2 of 64, 8 / 1 of 256
(window 512) and 8 / 1 of 512; vocabularies of 32000 and 262144.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

LAYOUTS = [(32, 8, 128, 0), (8, 2, 64, 0), (8, 1, 256, 512), (8, 1, 512, 0)]
DTYPE = {"f32": torch.float32, "f16": torch.float16}


def listed() -> list[dict]:
    return [
        # one decode step's append of one sequence: the smallest call
        dict(name="append_token", kind="append", dtype="f32", batch=1, heads=32, kv=8, hd=128, rotary=128, page=16, n=1, past=531,
             ragged=False),
        # one decode step's append of a serving batch
        dict(name="append_batch", kind="append", dtype="f16", batch=64, heads=32, kv=8, hd=128, rotary=128, page=64, n=1,
             past=4000, ragged=True),
        # padded prompts behind what each sequence already has, of which half the dims are rotated
        dict(name="append_prompts", kind="append", dtype="f16", batch=8, heads=32, kv=8, hd=128, rotary=64, page=32, n=2045,
             past=700, ragged=True),
        # one token's attention in a chat of a few hundred tokens
        dict(name="attn_chat", kind="attention", dtype="f32", batch=1, heads=32, kv=8, hd=128, n_q=1, page=16, len=531, shared=0,
             window=0, ragged=False),
        # one token of each sequence of a serving batch that shares nothing, lengths from none to 8 K
        dict(name="attn_batch", kind="attention", dtype="f16", batch=16, heads=32, kv=8, hd=128, n_q=1, page=64, len=8223,
             shared=0, window=0, ragged=True),
        # a batch behind a system prompt of 4 K, each with up to a few hundred tokens of its own
        dict(name="attn_prefix", kind="attention", dtype="f32", batch=32, heads=32, kv=8, hd=128, n_q=1, page=32, len=4810,
             shared=4096, window=0, ragged=True),
        # a large batch over one long document
        dict(name="attn_document", kind="attention", dtype="f16", batch=64, heads=32, kv=8, hd=128, n_q=1, page=128, len=17000,
             shared=16384, window=0, ragged=True),
        # drafts of five tokens checked at once, the shared part ending inside a page
        dict(name="attn_draft", kind="attention", dtype="f16", batch=8, heads=8, kv=2, hd=64, n_q=5, page=16, len=3001,
             shared=2003, window=0, ragged=True),
        # a sliding-window layer, whose window begins in the shared part for some sequences
        dict(name="attn_window", kind="attention", dtype="f32", batch=8, heads=8, kv=1, hd=256, n_q=1, page=32, len=4096,
             shared=3200, window=512, ragged=True),
        # the next token of one sequence, all filters on: the smallest call
        dict(name="sample_token", kind="sample", rows=1, n=32000, temperature=0.8, top_k=50, top_p=0.95, min_p=0.05, mixed=False,
             masked=0.0),
        # a serving batch whose users each chose their own filters
        dict(name="sample_batch", kind="sample", rows=256, n=32000, temperature=0.8, top_k=0, top_p=1.0, min_p=0.0, mixed=True,
             masked=0.01),
        # a few rows of the large vocabulary, by top-p alone
        dict(name="sample_vocab", kind="sample", rows=8, n=262144, temperature=1.0, top_k=0, top_p=0.9, min_p=0.0, mixed=False,
             masked=0.0),
    ]


def _log_uniform(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "attention", "attention", "sample"])
    if kind == "sample":
        n = rng.choice([32000, 262144, _log_uniform(rng, 2, 262144)])
        rows = _log_uniform(rng, 1, min(256, 256 * 32000 // n))
        return dict(kind=kind, rows=rows, n=n, temperature=rng.choice([0.0, 1.0, round(rng.uniform(0.2, 1.6), 3)]),
                    top_k=rng.choice([0, _log_uniform(rng, 1, n)]), top_p=rng.choice([1.0, round(rng.uniform(0.05, 0.999), 4)]),
                    min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]), mixed=rng.random() < 0.5,
                    masked=rng.choice([0.0, 0.01, 0.9]))
    heads, kv, hd, window = rng.choice(LAYOUTS)
    dtype, page = rng.choice(["f32", "f16"]), rng.choice([16, 32, 64, 128, 256])
    batch = _log_uniform(rng, 1, 64)
    # (each bounds a case by the largest listed one)
    if kind == "append":
        most = 2 ** 25 // (batch * heads * hd)
        return dict(kind=kind, dtype=dtype, batch=batch, heads=heads, kv=kv, hd=hd, rotary=rng.choice([hd, hd // 2]), page=page,
                    n=rng.choice([1, _log_uniform(rng, 1, min(2048, most))]),
                    past=rng.choice([0, _log_uniform(rng, 1, 4096)]), ragged=rng.random() < 0.5)
    n_q = rng.choice([1, 1, _log_uniform(rng, 1, 16)])
    tail = _log_uniform(rng, 1, min(16384, 2 ** 24 // (batch * kv * hd * n_q)))
    shared = rng.choice([0, _log_uniform(rng, 1, 16384 // n_q)])
    return dict(kind=kind, dtype=dtype, batch=batch, heads=heads, kv=kv, hd=hd, n_q=n_q, page=page, len=shared + tail,
                shared=shared, window=rng.choice([0, window]), ragged=rng.random() < 0.5)


def _lengths(case: dict, top: int, least: int = 0) -> list[int]:
    """The lengths of the batch's sequences: all `top`, or spread from `least` to `top`."""
    b = case["batch"]
    if not case["ragged"] or b == 1:
        return [top] * b
    return [least + round((top - least) * ((37 * i + 3) % b) / (b - 1)) for i in range(b)]


def work(case: dict) -> dict:
    if case["kind"] == "sample":
        cells = case["rows"] * case["n"]
        return {"bytes": 4 * cells + 28 * case["rows"], "flops": 2 * cells}
    heads, kv, hd, size = case["heads"], case["kv"], case["hd"], DTYPE[case["dtype"]].itemsize
    if case["kind"] == "append":
        rows = sum(_lengths(case, case["n"], 1))
        return {"bytes": rows * hd * (heads * 8 + 2 * kv * (4 + size)), "flops": rows * 3 * case["rotary"] * (heads + kv)}
    n_q, window, shared = case["n_q"], case["window"], case["shared"]
    lens = _lengths(case, case["len"], shared)
    first = [max(0, n - (window + n_q - 1)) if window else 0 for n in lens]
    seen = [n - lo for n, lo in zip(lens, first)]
    once = max([0] + [shared - lo for lo in first])
    rows = once + sum(n - max(lo, shared) for n, lo in zip(lens, first))
    return {"bytes": rows * kv * 2 * hd * size + case["batch"] * n_q * heads * hd * 8, "flops": 4 * hd * heads * n_q * sum(seen)}


# ---- inputs ---------------------------------------------------------------------------------------


def _rows(g, shape, keys: bool) -> torch.Tensor:
    """K or V rows [..., hd]: channels of different size, for keys a few large ones."""
    x = torch.randn(shape, generator=g, device=g.device)
    x *= torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=g.device))
    if keys:
        x[..., torch.randint(0, shape[-1], (3,), generator=g, device=g.device)] *= 6
    return x


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(s: dict, case: dict, g, slots: int, shared: int) -> None:
    """A pool in which every sequence has pages for `slots` entries, in no order; the whole pages among the first `shared`
    entries are the same ones for all."""
    b, page = case["batch"], case["page"]
    s["max_pages"], common = -(-slots // page), shared // page
    n_pages = common + b * (s["max_pages"] - common) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda")
    table = torch.cat([order[:common].expand(b, common), order[common:n_pages - 3].view(b, -1)], 1)
    s["table"] = table.int().contiguous()
    s["k"], s["v"] = (_rows(g, (n_pages, case["kv"], page, case["hd"]), keys).to(DTYPE[case["dtype"]]) for keys in (True, False))
    s["shared_pages"] = s["table"][0, :-(-shared // page)].clone()
    if own:
        from inference_engine_rust_amd import engine

        s["engine"] = engine
        s["cache"] = engine.PagedKV({"f32": engine.F32, "f16": engine.F16}[case["dtype"]], n_pages, case["kv"], page, case["hd"],
                                    s["k"].data_ptr(), s["v"].data_ptr(), b, s["max_pages"], s["table"].data_ptr())


def _prepare_append(case: dict, g) -> dict:
    s = dict(case)
    b, heads, kv, hd, n, rotary = (case[x] for x in ("batch", "heads", "kv", "hd", "n", "rotary"))
    s["stride"] = (heads + 2 * kv) * hd
    s["rows"] = torch.randn((b, n, s["stride"]), generator=g, device="cuda") * 1.5
    s["start"], s["count"] = _ints(_lengths(case, case["past"])[::-1]), _ints(_lengths(case, n, 1))
    _pages(s, case, g, case["past"] + n, 0)
    places = s["max_pages"] * case["page"]
    pair = torch.arange(rotary // 2, dtype=torch.float64, device="cuda")
    angle = torch.arange(places, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-2 * pair / rotary)
    s["rope"] = torch.stack([angle.cos(), angle.sin()], 2).float()
    s["q_out"] = torch.zeros((b, n, heads, hd), device="cuda")
    s["len_out"] = _ints([0] * b)
    return s


def _prepare_attention(case: dict, g) -> dict:
    s = dict(case)
    b, heads, kv, hd, n_q = (case[x] for x in ("batch", "heads", "kv", "hd", "n_q"))
    _pages(s, case, g, case["len"] + 1, case["shared"])
    s["lens"], s["shared_len"] = _ints(_lengths(case, case["len"], case["shared"])), _ints([case["shared"]])
    s["stride"] = (heads + 2 * kv) * hd  # rows of a fused q / k / v projection
    s["q"] = torch.randn((b, n_q, s["stride"]), generator=g, device="cuda") * 1.5
    s["scale"] = 1 / math.sqrt(hd)
    s["out"] = torch.zeros((b, n_q, heads, hd), device="cuda")
    # the page that the shared part ends in is each sequence's own: its first entries are copies
    page, cut = case["page"], case["shared"] % case["page"]
    if cut:
        last = s["table"][:, case["shared"] // page].long()
        for pool in (s["k"], s["v"]):
            pool[last, :, :cut] = pool[last[:1], :, :cut]
    if own:
        size = s["engine"].paged_attention_workspace(s["cache"], heads, n_q, case["len"], case["shared"])
        s["ws"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    return s


def _prepare_sample(case: dict, g) -> dict:
    s = dict(case)
    rows, n = case["rows"], case["n"]

    def uniform(lo=0.0, hi=1.0):
        return lo + (hi - lo) * torch.rand(rows, generator=g, device="cuda")

    # a bulk, and a few dozen likely tokens a row
    logits = torch.randn((rows, n), generator=g, device="cuda") * 2
    logits += 7 * torch.relu(torch.randn((rows, n), generator=g, device="cuda") - 2.5)
    if case["masked"]:  # tokens that a grammar forbids
        banned = torch.rand((rows, n), generator=g, device="cuda") < case["masked"]
        banned[:, n // 2] = False
        logits.masked_fill_(banned, -math.inf)
    s["logits"] = logits
    s["temperature_rows"] = torch.full((rows,), case["temperature"], device="cuda")
    s["top_k_rows"] = torch.full((rows,), case["top_k"], dtype=torch.int32, device="cuda")
    s["top_p_rows"] = torch.full((rows,), case["top_p"], device="cuda")
    s["min_p_rows"] = torch.full((rows,), case["min_p"], device="cuda")
    if case["mixed"]:
        s["temperature_rows"] = torch.where(uniform() < 0.15, torch.zeros(()).cuda(), uniform(0.3, 1.5))
        s["top_k_rows"] = torch.where(uniform() < 0.5, torch.zeros(()).cuda(), uniform(1, 200)).int()
        s["top_p_rows"] = torch.where(uniform() < 0.4, torch.ones(()).cuda(), uniform(0.3, 0.99))
        s["min_p_rows"] = torch.where(uniform() < 0.6, torch.zeros(()).cuda(), uniform(0.01, 0.2))
    s["r"] = uniform()
    s["index"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
    s["prob"] = torch.zeros(rows, device="cuda")
    if own:
        from inference_engine_rust_amd import engine

        s["engine"] = engine
        s["ws"] = torch.empty(max(engine.sample_workspace(rows, n), 1), dtype=torch.uint8, device="cuda")
    return s


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"append": _prepare_append, "attention": _prepare_attention, "sample": _prepare_sample}[case["kind"]](case, g)


# ---- the operators ----------------------------------------------------------------------------------


def _rotated(x: torch.Tensor, rope: torch.Tensor) -> torch.Tensor:
    """Rows [..., heads, hd] with the adjacent pairs of their first dims turned by rope [..., pairs, 2]."""
    pairs = rope.shape[-2]
    a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
    c, s = rope[..., None, :, 0], rope[..., None, :, 1]
    turned = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * pairs:]], -1)


def _append_plain(s: dict):
    b, heads, kv, hd, n, page = (s[x] for x in ("batch", "heads", "kv", "hd", "n", "page"))
    i = torch.arange(n, device="cuda")
    live = i < s["count"][:, None]
    at = torch.where(live, s["start"].long()[:, None] + i, 0)
    x = s["rows"].view(b, n, heads + 2 * kv, hd)
    turned = _rotated(x[:, :, :heads + kv], s["rope"][at])
    q = torch.where(live[..., None, None], turned[:, :, :heads], 0)
    where, slot = torch.gather(s["table"].long(), 1, at // page)[live], (at % page)[live]
    s["k"][where, :, slot] = turned[:, :, heads:][live].to(s["k"].dtype)
    s["v"][where, :, slot] = x[:, :, heads + kv:][live].to(s["v"].dtype)
    return dict(q=q, k=s["k"], v=s["v"], len=s["start"] + s["count"])


def _gathered(pool: torch.Tensor, pages: torch.Tensor, lo: int, hi: int) -> torch.Tensor:
    """Entries lo .. hi of the sequences whose pages [..., max_pages] are given, [..., n_kv, hi - lo, hd] in f32."""
    page, first = pool.shape[2], lo // pool.shape[2]
    x = pool[pages[..., first:-(-hi // page)].long()].transpose(-4, -3).flatten(-3, -2)
    return x[..., lo - first * page:hi - first * page, :].float()


def _attention_plain(s: dict):
    b, heads, kv, hd, n_q, n, shared = (s[x] for x in ("batch", "heads", "kv", "hd", "n_q", "len", "shared"))
    group = heads // kv
    q = s["q"][..., :heads * hd].view(b, n_q, kv, group, hd).permute(2, 0, 1, 3, 4) * s["scale"]
    # the shared entries for all columns at once, then each sequence's own
    keys, values = (_gathered(pool, s["shared_pages"], 0, shared) for pool in (s["k"], s["v"]))
    scores = torch.matmul(q.reshape(kv, b * n_q * group, hd), keys.transpose(-2, -1).contiguous()).view(kv, b, n_q * group, shared)
    keys, own_values = (_gathered(pool, s["table"], shared, n).transpose(0, 1) for pool in (s["k"], s["v"]))
    more = torch.matmul(q.reshape(kv, b, -1, hd), keys.transpose(-2, -1).contiguous())
    scores = torch.cat([scores, more], -1).view(kv, b, n_q, group, n)
    j = torch.arange(n, device="cuda")
    limit = s["lens"].long()[:, None] - torch.arange(n_q - 1, -1, -1, device="cuda")
    seen = j < limit[..., None]
    if s["window"]:
        seen &= j >= limit[..., None] - s["window"]
    scores.masked_fill_(~seen[:, :, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-3e38))
    p = (p / p.sum(-1, keepdim=True).clamp_min(1e-38)).view(kv, b, -1, n)
    out = torch.matmul(p[..., shared:], own_values.contiguous())
    out += torch.matmul(p[..., :shared].reshape(kv, b * n_q * group, shared), values).view(kv, b, -1, hd)
    return dict(out=out.view(kv, b, n_q, group, hd).permute(1, 2, 0, 3, 4).reshape(b, n_q, heads, hd))


def _sample_plain(s: dict):
    x, n = s["logits"], s["n"]
    top = x.amax(1, keepdim=True)
    greedy = s["temperature_rows"][:, None] == 0
    t = torch.where(greedy, 1, s["temperature_rows"][:, None]).double()
    order = torch.argsort(x, dim=1, descending=True, stable=True)
    w = torch.exp((x.double() - top.double()) / t)
    ranked = torch.gather(w, 1, order)
    rank = torch.arange(n, device="cuda")
    k = torch.where((s["top_k_rows"] > 0) & ~greedy[:, 0], s["top_k_rows"], n)[:, None]
    k = torch.where(greedy, 1, k)
    ranked = torch.where(rank < k, ranked, 0)
    upto = torch.cumsum(ranked, 1)
    p = s["top_p_rows"][:, None].double()
    keep = (rank < k) & ((p >= 1) | (upto - ranked < p * upto[:, -1:]))
    keep &= ranked >= s["min_p_rows"][:, None].double()
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ranked, 0))
    upto = torch.cumsum(kept, 1)
    total = upto[:, -1:]
    index = (upto <= s["r"][:, None].double() * total).sum(1, keepdim=True)
    return dict(index=index[:, 0].int(), prob=(torch.gather(kept, 1, index) / total)[:, 0].float())


def run(s: dict):
    if not own:
        return {"append": _append_plain, "attention": _attention_plain, "sample": _sample_plain}[s["kind"]](s)
    engine = s["engine"]
    stream = torch.cuda.current_stream().cuda_stream
    if s["kind"] == "append":
        heads, kv, hd = s["heads"], s["kv"], s["hd"]
        q = s["rows"].data_ptr()
        k = q + 4 * heads * hd
        engine.paged_append(s["cache"], q, k, k + 4 * kv * hd, heads, s["n"], s["stride"], s["rope"].data_ptr(),
                            s["rope"].shape[0], s["rotary"], s["start"].data_ptr(), s["count"].data_ptr(),
                            s["len_out"].data_ptr(), s["q_out"].data_ptr(), heads * hd, stream)
        return dict(q=s["q_out"], k=s["k"], v=s["v"], len=s["len_out"])
    if s["kind"] == "attention":
        engine.paged_attention(s["cache"], s["q"].data_ptr(), s["heads"], s["n_q"], s["stride"], s["lens"].data_ptr(), s["len"],
                               s["shared_pages"].data_ptr(), s["shared_len"].data_ptr(), s["shared"], s["window"], s["scale"],
                               s["out"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(), stream)
        return dict(out=s["out"])
    engine.sample(s["logits"].data_ptr(), s["rows"], s["n"], s["n"], s["temperature_rows"].data_ptr(),
                  s["top_k_rows"].data_ptr(), s["top_p_rows"].data_ptr(), s["min_p_rows"].data_ptr(), s["r"].data_ptr(),
                  s["index"].data_ptr(), s["prob"].data_ptr(), s["ws"].data_ptr(), s["ws"].numel(), stream)
    return dict(index=s["index"], prob=s["prob"])


# ---- the definitions in 64 bits ---------------------------------------------------------------------


def _exact_append(case: dict, s: dict):
    heads, kv, page, pairs = case["heads"], case["kv"], case["page"], case["rotary"] // 2
    k, v = s["k"].double(), s["v"].double()
    q = torch.zeros(s["q_out"].shape, dtype=torch.float64, device="cuda")
    for b, (start, count) in enumerate(zip(s["start"].tolist(), s["count"].tolist())):
        x = s["rows"][b, :count].double().view(count, heads + 2 * kv, case["hd"])
        pos = torch.arange(start, start + count, device="cuda")
        spin = torch.complex(s["rope"][pos, :, 0].double(), s["rope"][pos, :, 1].double())[:, None]
        x[:, :heads + kv, :2 * pairs] = torch.view_as_real(
            torch.view_as_complex(x[:, :heads + kv, :2 * pairs].reshape(count, heads + kv, pairs, 2)) * spin).flatten(2)
        q[b, :count] = x[:, :heads]
        where = s["table"][b].long()[pos // page]
        k[where, :, pos % page], v[where, :, pos % page] = x[:, heads:heads + kv], x[:, heads + kv:]
    return dict(q=q, k=k, v=v, len=None)


def _exact_attention(case: dict, s: dict):
    heads, kv, hd, n_q, page = (case[x] for x in ("heads", "kv", "hd", "n_q", "page"))
    out = torch.zeros((case["batch"], n_q, heads, hd), dtype=torch.float64, device="cuda")
    group = heads // kv
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, :-(-n // page)].long()
        for h in range(kv):
            keys, values = (pool[pages, h].flatten(0, 1)[:n].double() for pool in (s["k"], s["v"]))
            for t in range(n_q):
                hi = n - (n_q - 1 - t)
                lo = max(0, hi - case["window"]) if case["window"] else 0
                if hi > lo:
                    q = s["q"][b, t, h * group * hd:(h + 1) * group * hd].double().view(group, hd)
                    p = torch.softmax(keys[lo:hi] @ q.t().contiguous() * s["scale"], 0)
                    out[b, t, h * group:(h + 1) * group] = p.t().contiguous() @ values[lo:hi]
    return dict(out=out)


def _exact_sample(case: dict, s: dict):
    names = ("temperature_rows", "top_k_rows", "top_p_rows", "min_p_rows", "r")
    probs = []
    for x, t, k, p, least, r in zip(s["logits"].double().cpu().numpy(), *(s[a].double().cpu().numpy() for a in names)):
        if t == 0:
            probs.append(1.0)
            continue
        order = np.argsort(-x, kind="stable")
        order = order[:int(k)] if 0 < k < len(order) else order
        w = np.exp((x[order] - x[order[0]]) / t)
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        kept = (w >= least) & ((before < p * w.sum()) if p < 1 else True)
        chosen = np.sort(order[kept])
        w = np.exp((x[chosen] - x[order[0]]) / t)
        i = np.searchsorted(np.cumsum(w), r * w.sum(), side="right")
        probs.append(w[i] / w.sum())
    return dict(index=None, prob=np.array(probs))


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[case["kind"]](case, s)
