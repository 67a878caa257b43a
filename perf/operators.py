"""The operators of the 8-bit KV cache: append, attention, eviction, in a plain form and as the framework's calls.

The cache holds keys and values as 8-bit codes (int8, or e4m3) of shape [batch][n_kv][capacity][head_dim] and a
power-of-two f32 scale for each block of 32 slots of a head. Kinds of case:

* ``append``  — new K / V rows (f32, a slice of fused rows) into the cache, and the touched blocks read back as the values
  they now stand for.
* ``attention``  — the query rows of one or several new tokens per sequence over the cache, optionally adding each entry's
  attention weight to its running sum.
* ``evict``  — a cache cut down to the entries of the largest running weight, in another, smaller cache, and that read back.

Head layouts are those of the repository's configurations: 32 heads / 8 KV heads of 128, 8 / 2 of 64, 8 / 1 of 256
(window 512) and 8 / 1 of 512.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = 32
TOP = {"i8": 127.0, "e4m3": 448.0}
LAYOUTS = [(32, 8, 128, 0), (8, 2, 64, 0), (8, 1, 256, 512), (8, 1, 512, 0)]


def listed() -> list[dict]:
    return [
        # one decode step's append of one sequence: the smallest call
        dict(name="append_token", kind="append", dtype="i8", batch=1, kv=8, hd=128, n=1, past=531, ragged=False),
        # one decode step's append of a serving batch
        dict(name="append_batch", kind="append", dtype="e4m3", batch=32, kv=8, hd=128, n=1, past=4000, ragged=True),
        # a 2-K prompt of odd length into an empty cache
        dict(name="append_prompt", kind="append", dtype="i8", batch=1, kv=8, hd=128, n=2045, past=0, ragged=False),
        # chunks of padded prompts behind what each sequence already has
        dict(name="append_chunks", kind="append", dtype="e4m3", batch=8, kv=2, hd=64, n=4096, past=700, ragged=True),
        # one token's attention in a chat of a few hundred tokens
        dict(name="attn_chat", kind="attention", dtype="i8", batch=1, heads=32, kv=8, hd=128, n_q=1, len=531, window=0,
             weights=False, ragged=False),
        # one token over a long context that is about to be evicted from
        dict(name="attn_long", kind="attention", dtype="i8", batch=1, heads=32, kv=8, hd=128, n_q=1, len=32768, window=0,
             weights=True, ragged=False),
        # one token of each sequence of a serving batch, lengths from none to 8 K
        dict(name="attn_batch", kind="attention", dtype="e4m3", batch=16, heads=32, kv=8, hd=128, n_q=1, len=8223,
             window=0, weights=False, ragged=True),
        # a draft of five tokens checked at once
        dict(name="attn_draft", kind="attention", dtype="e4m3", batch=4, heads=8, kv=2, hd=64, n_q=5, len=3001, window=0,
             weights=False, ragged=True),
        # a sliding-window layer of a batch
        dict(name="attn_window", kind="attention", dtype="i8", batch=8, heads=8, kv=1, hd=256, n_q=1, len=4096, window=512,
             weights=True, ragged=True),
        # a chat that passed its budget
        dict(name="evict_chat", kind="evict", dtype="i8", batch=1, kv=8, hd=128, len=1157, keep=1024, first=4, last=128,
             ragged=False),
        # long prompts cut down before decoding
        dict(name="evict_long", kind="evict", dtype="i8", batch=4, kv=8, hd=128, len=32768, keep=8192, first=4, last=1024,
             ragged=True),
        # a wide single KV head
        dict(name="evict_wide", kind="evict", dtype="e4m3", batch=4, kv=1, hd=512, len=8223, keep=3000, first=1, last=333,
             ragged=True),
    ]


def _log_uniform(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    heads, kv, hd, window = rng.choice(LAYOUTS)
    kind = rng.choice(["append", "attention", "attention", "evict"])
    dtype = rng.choice(["i8", "e4m3"])
    batch = _log_uniform(rng, 1, 32)
    most = 2 ** 28 // (batch * kv * hd)  # bounds a case by the largest listed one
    if kind == "append":
        n = rng.choice([1, _log_uniform(rng, 1, max(2, min(4096, most // 16)))])
        return dict(kind=kind, dtype=dtype, batch=batch, kv=kv, hd=hd, n=n, past=rng.choice([0, _log_uniform(rng, 1, 8704)]),
                    ragged=rng.random() < 0.5)
    n_q = rng.choice([1, 1, _log_uniform(rng, 1, 16)]) if kind == "attention" else 1
    length = _log_uniform(rng, 1, min(32768, most // (4 * n_q)))
    ragged = rng.random() < 0.5
    if kind == "attention":
        return dict(kind=kind, dtype=dtype, batch=batch, heads=heads, kv=kv, hd=hd, n_q=n_q, len=length,
                    window=rng.choice([0, window]), weights=rng.random() < 0.5, ragged=ragged)
    keep = min(_log_uniform(rng, 1, length), most // 16)
    first = rng.randint(0, min(4, keep))
    return dict(kind=kind, dtype=dtype, batch=batch, kv=kv, hd=hd, len=length, keep=keep, first=first,
                last=rng.randint(0, keep - first), ragged=ragged)


def _lengths(case: dict, top: int, least: int = 0) -> list[int]:
    """The lengths of the batch's sequences: all `top`, or spread from `least` to `top`."""
    b = case["batch"]
    if not case["ragged"] or b == 1:
        return [top] * b
    return [least + round((top - least) * ((37 * i + 3) % b) / (b - 1)) for i in range(b)]


def work(case: dict) -> dict:
    kv, hd = case["kv"], case["hd"]
    if case["kind"] == "append":
        rows = sum(_lengths(case, case["n"], 1)) * kv
        return {"bytes": rows * 2 * hd * (4 + 1 + 4), "flops": rows * 2 * hd * 2}
    lens = _lengths(case, case["len"])
    if case["kind"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lens) * kv
        return {"bytes": sum(lens) * kv * 4 + kept * (2 * hd * (1 + 1 + 4) + 8), "flops": kept * 2 * hd}
    heads, n_q, window = case["heads"], case["n_q"], case["window"]
    seen = [n if not window else min(n, window + n_q - 1) for n in lens]
    return {"bytes": sum(seen) * kv * (2 * hd + 8 / BLOCK + (8 if case["weights"] else 0)) + case["batch"] * n_q * heads * hd * 8,
            "flops": 4 * hd * heads * n_q * sum(seen)}


# ---- inputs ---------------------------------------------------------------------------------------


def _rows(g, shape, keys: bool) -> torch.Tensor:
    """K or V rows [..., n, hd]: channels of different size, for keys a few large ones, for values small first tokens."""
    dev = g.device
    x = torch.randn(shape, generator=g, device=dev)
    x *= torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=dev))
    x *= torch.exp(0.3 * torch.randn(shape[:-1], generator=g, device=dev))[..., None]
    if keys:
        x[..., torch.randint(0, shape[-1], (3,), generator=g, device=dev)] *= 6
    else:
        x[..., :4, :] *= 0.1
    return x


def _pow2_scale(amax: torch.Tensor, dtype: str) -> torch.Tensor:
    """The smallest power of two s >= 2^-100 with amax <= TOP * s."""
    mant, exp = torch.frexp(amax)
    top_mant, top_exp = math.frexp(TOP[dtype])
    e = exp - top_exp + (mant > top_mant).int()
    return torch.ldexp(torch.ones_like(amax), e.clamp_min(-100) * (amax > 0) - 100 * (amax <= 0).int())


def _round(x: torch.Tensor, dtype: str) -> torch.Tensor:
    """Values in units of the scale, rounded to the codes' values (f32)."""
    return torch.round(x) if dtype == "i8" else x.to(torch.float8_e4m3fn).float()


def _codes(x: torch.Tensor, dtype: str) -> torch.Tensor:
    return x.to(torch.int8) if dtype == "i8" else x.to(torch.float8_e4m3fn)


def _filled(g, case: dict, cap: int, keys: bool):
    """Codes [batch][kv][cap][hd] and scales [batch][kv][ceil(cap / 32)] of a cache full of rows."""
    b, kv, hd = case["batch"], case["kv"], case["hd"]
    nb = -(-cap // BLOCK)
    codes, scales = [], []
    for _ in range(b):
        x = _rows(g, (kv, nb * BLOCK, hd), keys)
        s = _pow2_scale(x.view(kv, nb, BLOCK * hd).abs().amax(2), case["dtype"])
        y = _round(x.view(kv, nb, BLOCK, hd) / s[:, :, None, None], case["dtype"])
        codes.append(_codes(y.view(kv, nb * BLOCK, hd)[:, :cap], case["dtype"]))
        scales.append(s)
    return torch.stack(codes), torch.stack(scales)


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(s: dict, case: dict, codes_scales, cap: int, name: str = "cache") -> None:
    (s["kc"], s["ks"]), (s["vc"], s["vs"]) = codes_scales
    _handle(s, name, case, cap, s["kc"], s["vc"], s["ks"], s["vs"])


def _handle(s: dict, name: str, case: dict, cap: int, kc, vc, ks, vs) -> None:
    """The descriptor that a program keeps beside its buffers."""
    if own:
        from inference_engine_rust_amd import engine

        s["engine"] = engine
        s[name] = engine.KV8Cache({"i8": engine.I8, "e4m3": engine.E4M3}[case["dtype"]], case["batch"], case["kv"], cap,
                                  case["hd"], kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr())


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    b, kv, hd = case["batch"], case["kv"], case["hd"]
    f32 = dict(dtype=torch.float32, device="cuda")
    if case["kind"] == "append":
        n = case["n"]
        counts, starts = _lengths(case, n, 1), _lengths(case, case["past"])[::-1]
        cap = -(-(case["past"] + n) // BLOCK) * BLOCK + 2 * BLOCK
        _cache(s, case, [_filled(g, case, cap, True), _filled(g, case, cap, False)], cap)
        rows = torch.cat([_rows(g, (b, kv, n, hd), keys).transpose(1, 2).reshape(b, n, kv * hd) for keys in (True, False)], 2)
        s.update(rows=rows, start=_ints(starts), count=_ints(counts), len_out=_ints([0] * b))
        # the touched blocks: from the start of the first to the last new row
        s["span"] = (-(-n // BLOCK) + 1) * BLOCK
        s["span_start"] = _ints([x // BLOCK * BLOCK for x in starts])
        s["span_count"] = _ints([x % BLOCK + c for x, c in zip(starts, counts)])
        s["out_k"], s["out_v"] = (torch.zeros((b, s["span"], kv, hd), **f32) for _ in range(2))
        return s
    lens = _lengths(case, case["len"])
    s["lens"] = _ints(lens)
    cap = case["len"] + 33
    _cache(s, case, [_filled(g, case, cap, True), _filled(g, case, cap, False)], cap)
    s["nb"] = s["ks"].shape[2]
    weights = torch.exp(2.5 * torch.randn((b, kv, cap), generator=g, device="cuda") - 6)
    weights *= torch.rand((b, kv, cap), generator=g, device="cuda") > 0.02  # entries that no query has seen
    if case["kind"] == "attention":
        heads, n_q = case["heads"], case["n_q"]
        s["stride"] = (heads + 2 * kv) * hd  # rows of a fused q / k / v projection
        s["fused"] = torch.randn((b, n_q, s["stride"]), generator=g, device="cuda") * 1.5
        s["scale"] = 1 / math.sqrt(hd)
        s["out"] = torch.zeros((b, n_q, heads, hd), **f32)
        s["weights_in"], s["weights_out"] = weights, torch.zeros_like(weights)
        if own:
            size = s["engine"].kv8_attention_workspace(s["cache"], heads, n_q, case["len"], case["weights"])
            s["ws"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
        return s
    keep = case["keep"]
    s["weights_in"] = weights
    s["to_cap"] = keep + 40
    s["to_kc"], s["to_vc"] = (torch.zeros((b, kv, s["to_cap"], hd), dtype=s["kc"].dtype, device="cuda") for _ in range(2))
    s["to_ks"], s["to_vs"] = (torch.ones((b, kv, -(-s["to_cap"] // BLOCK)), **f32) for _ in range(2))
    s["weights_out"] = torch.zeros((b, kv, s["to_cap"]), **f32)
    s["index"] = torch.zeros((b, kv, keep), dtype=torch.int32, device="cuda")
    s["len_out"] = _ints([0] * b)
    s["out_k"], s["out_v"] = (torch.zeros((b, keep, kv, hd), **f32) for _ in range(2))
    _handle(s, "to", case, s["to_cap"], s["to_kc"], s["to_vc"], s["to_ks"], s["to_vs"])
    if own:
        size = s["engine"].kv8_evict_workspace(s["cache"], case["len"], keep)
        s["ws"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    return s


# ---- the operators ----------------------------------------------------------------------------------


def _append_plain(s: dict):
    b, kv, hd, n, span = s["batch"], s["kv"], s["hd"], s["n"], s["span"]
    nb = span // BLOCK
    start, count = s["start"].long(), s["count"].long()
    r = torch.arange(span, device="cuda")
    i = r - (start % BLOCK)[:, None]  # index of the new row at each place of the span
    new, old = (i >= 0) & (i < count[:, None]), (i < 0)[:, :BLOCK]
    seq = torch.arange(b, device="cuda")[:, None]
    blocks = (start // BLOCK)[:, None] + torch.arange(nb, device="cuda")
    inside = blocks.clamp_max(s["ks"].shape[2] - 1)
    touched = new.view(b, nb, BLOCK).any(2)[:, None, :]
    first = (blocks[:, :1] * BLOCK + r[:BLOCK]).clamp_max(s["kc"].shape[2] - 1)
    outputs = []
    for x, codes, scales in ((s["rows"][..., :kv * hd], s["kc"], s["ks"]), (s["rows"][..., kv * hd:], s["vc"], s["vs"])):
        x = torch.where(new[..., None], x[seq, i.clamp(0, n - 1)], 0).view(b, span, kv, hd)
        scale = _pow2_scale(x.abs().view(b, nb, BLOCK, kv, hd).amax((2, 4)), s["dtype"]).transpose(1, 2)
        before = scales[seq, :, inside].transpose(1, 2)
        scale[..., 0] = torch.where((start % BLOCK > 0)[:, None], torch.maximum(scale[..., 0], before[..., 0]), scale[..., 0])
        each = scale.transpose(1, 2).repeat_interleave(BLOCK, 1)[..., None]
        value = _round(x / each, s["dtype"]) * each
        kept = _round(codes[seq, :, first].float() * (before / scale)[:, None, :, :1], s["dtype"]) * scale[:, None, :, :1]
        value[:, :BLOCK] = torch.where(old[:, :, None, None], kept, value[:, :BLOCK])
        after = scales.clone()
        after[seq, :, inside] = torch.where(touched, scale, before).transpose(1, 2)
        outputs += [value, after]
    return dict(k=outputs[0], v=outputs[2], k_scale=outputs[1], v_scale=outputs[3], len=(start + count).int())


def _values(codes: torch.Tensor, scales: torch.Tensor, n: int) -> torch.Tensor:
    return codes[:, :, :n].float() * scales.repeat_interleave(BLOCK, 2)[:, :, :n, None]


def _attention_plain(s: dict):
    b, kv, hd, n_q, heads, n = s["batch"], s["kv"], s["hd"], s["n_q"], s["heads"], s["len"]
    q = s["fused"][..., :heads * hd].view(b, n_q, kv, heads // kv, hd).permute(0, 2, 1, 3, 4).reshape(b, kv, -1, hd)
    scores = torch.matmul(q * s["scale"], _values(s["kc"], s["ks"], n).transpose(2, 3)).view(b, kv, n_q, -1, n)
    j = torch.arange(n, device="cuda")
    limit = s["lens"].long()[:, None] - torch.arange(n_q - 1, -1, -1, device="cuda")
    seen = j < limit[..., None]
    if s["window"]:
        seen &= j >= limit[..., None] - s["window"]
    seen = seen[:, None, :, None]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(scores - top)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-38)
    out = torch.matmul(p.view(b, kv, -1, n), _values(s["vc"], s["vs"], n)).view(b, kv, n_q, -1, hd)
    out = out.permute(0, 2, 1, 3, 4).reshape(b, n_q, heads, hd)
    if not s["weights"]:
        return dict(out=out)
    total = torch.zeros_like(s["weights_in"])
    total[..., :n] = torch.where((j < s["lens"][:, None])[:, None], s["weights_in"][..., :n] + p.sum((2, 3)), 0)
    return dict(out=out, weights=total)


def _evict_plain(s: dict):
    b, kv, hd, n, keep = s["batch"], s["kv"], s["hd"], s["len"], s["keep"]
    lens = s["lens"].long()[:, None, None]
    j = torch.arange(n, device="cuda")
    key = torch.where((j < s["first"]) | (j >= lens - s["last"]), math.inf, s["weights_in"][..., :n])
    key = torch.where(j < lens, key, -math.inf)
    order = torch.argsort(key, dim=2, descending=True, stable=True)[..., :keep]
    index = torch.sort(torch.where(torch.gather((j < lens).expand(b, kv, n), 2, order), order, n), dim=2).values
    alive = index < n
    index = torch.where(alive, index, 0)
    out = dict(index=index.int(), len=s["lens"].clamp_max(keep))
    out["weights"] = torch.zeros_like(s["weights_out"])
    out["weights"][..., :keep] = torch.where(alive, torch.gather(s["weights_in"], 2, index), 0)
    nb = -(-keep // BLOCK)
    for name, codes, scales, fresh in (("k", s["kc"], s["ks"], s["to_ks"]), ("v", s["vc"], s["vs"], s["to_vs"])):
        from_scale = torch.where(alive, torch.gather(scales, 2, index // BLOCK), 0)
        padded = torch.nn.functional.pad(from_scale, (0, nb * BLOCK - keep))
        scale = padded.view(b, kv, nb, BLOCK).amax(3)
        each = scale.repeat_interleave(BLOCK, 2)[..., :keep, None].clamp_min(1e-38)
        rows = torch.gather(codes, 2, index[..., None].expand(b, kv, keep, hd)).float()
        value = torch.where(alive[..., None], _round(rows * (from_scale[..., None] / each), s["dtype"]) * each, 0)
        out[name] = value.transpose(1, 2).contiguous()
        out[name + "_scale"] = torch.ones_like(fresh)
        out[name + "_scale"][..., :nb] = torch.where(scale > 0, scale, 1)
    return out


def run(s: dict):
    if not own:
        return {"append": _append_plain, "attention": _attention_plain, "evict": _evict_plain}[s["kind"]](s)
    engine, kv, hd = s["engine"], s["kv"], s["hd"]
    stream = torch.cuda.current_stream().cuda_stream
    if s["kind"] == "append":
        k = s["rows"].data_ptr()
        engine.kv8_append(s["cache"], k, k + 4 * kv * hd, s["n"], 2 * kv * hd, s["start"].data_ptr(), s["count"].data_ptr(),
                          s["len_out"].data_ptr(), 0, stream)
        engine.kv8_load(s["cache"], s["span"], kv * hd, s["span_start"].data_ptr(), s["span_count"].data_ptr(),
                        s["out_k"].data_ptr(), s["out_v"].data_ptr(), stream)
        return dict(k=s["out_k"], v=s["out_v"], k_scale=s["ks"], v_scale=s["vs"], len=s["len_out"])
    if s["kind"] == "attention":
        w_in, w_out = (s["weights_in"].data_ptr(), s["weights_out"].data_ptr()) if s["weights"] else (0, 0)
        engine.kv8_attention(s["cache"], s["fused"].data_ptr(), s["heads"], s["n_q"], s["stride"], s["lens"].data_ptr(),
                             s["len"], s["window"], s["scale"], s["out"].data_ptr(), w_in, w_out, s["ws"].data_ptr(),
                             s["ws"].numel(), stream)
        return dict(out=s["out"], weights=s["weights_out"]) if s["weights"] else dict(out=s["out"])
    engine.kv8_evict(s["cache"], s["to"], s["weights_in"].data_ptr(), s["weights_out"].data_ptr(), s["lens"].data_ptr(),
                     s["len_out"].data_ptr(), s["len"], s["keep"], s["first"], s["last"], s["index"].data_ptr(),
                     s["ws"].data_ptr(), s["ws"].numel(), stream)
    engine.kv8_load(s["to"], s["keep"], kv * hd, 0, s["len_out"].data_ptr(), s["out_k"].data_ptr(), s["out_v"].data_ptr(),
                    stream)
    return dict(index=s["index"], len=s["len_out"], weights=s["weights_out"], k=s["out_k"], k_scale=s["to_ks"], v=s["out_v"],
                v_scale=s["to_vs"])


# ---- the definitions in 64 bits ---------------------------------------------------------------------


def _np_scale(amax: np.ndarray, top: float) -> np.ndarray:
    with np.errstate(divide="ignore"):
        return 2.0 ** np.maximum(np.ceil(np.log2(amax / top)), -100)


def _np_round(x: np.ndarray, dtype: str) -> np.ndarray:
    if dtype == "i8":
        return np.rint(x)
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -20))), -6) - 3)  # e4m3: three mantissa bits
    return np.rint(x / step) * step


def _np_append(case: dict, s: dict):
    top, n, kv, hd = TOP[case["dtype"]], case["n"], case["kv"], case["hd"]
    starts, counts = s["start"].tolist(), s["count"].tolist()
    rows = s["rows"].double().cpu().numpy().reshape(case["batch"], n, 2, kv, hd)
    got = {}
    for t, name, codes, scales in ((0, "k", s["kc"], s["ks"]), (1, "v", s["vc"], s["vs"])):
        scales = scales.double().cpu().numpy()
        values = np.zeros((case["batch"], s["span"], kv, hd))
        for b, (start, count) in enumerate(zip(starts, counts)):
            base = start - start % BLOCK
            for lo in range(base, start + count, BLOCK):
                here = rows[b, max(lo, start) - start:min(lo + BLOCK, start + count) - start, t]
                scale = _np_scale(np.abs(here).max((0, 2)), top)
                if lo < start:
                    was = scales[b, :, lo // BLOCK].copy()
                    scale = np.maximum(scale, was)
                    earlier = codes[b, :, lo:start].double().cpu().numpy().transpose(1, 0, 2)
                    values[b, :start - lo] = _np_round(earlier * (was / scale)[:, None], case["dtype"]) * scale[:, None]
                at = max(lo, start) - base
                values[b, at:at + len(here)] = _np_round(here / scale[:, None], case["dtype"]) * scale[:, None]
                scales[b, :, lo // BLOCK] = scale
        got[name], got[name + "_scale"] = values, scales
    return dict(k=got["k"], v=got["v"], k_scale=got["k_scale"], v_scale=got["v_scale"], len=None)


def _f64_attention(case: dict, s: dict):
    heads, kv, hd, n_q = case["heads"], case["kv"], case["hd"], case["n_q"]
    out = torch.zeros((case["batch"], n_q, heads, hd), dtype=torch.float64, device="cuda")
    weights = torch.zeros(s["weights_in"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lens"].tolist()):
        weights[b, :, :n] = s["weights_in"][b, :, :n]
        for h in range(kv):
            each = torch.arange(n, device="cuda") // BLOCK
            keys, vals = (c[b, h, :n].double() * x[b, h].double()[each][:, None] for c, x in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
            group = slice(h * (heads // kv), (h + 1) * (heads // kv))
            for t in range(n_q):
                hi = n - (n_q - 1 - t)
                lo = max(0, hi - case["window"]) if case["window"] else 0
                if hi <= lo:
                    continue
                q = s["fused"][b, t, :heads * hd].double().view(heads, hd)[group]
                p = torch.softmax(keys[lo:hi] @ q.t().contiguous() * s["scale"], 0)
                out[b, t, group] = p.t().contiguous() @ vals[lo:hi]
                weights[b, h, lo:hi] += p.sum(1)
    return dict(out=out, weights=weights) if case["weights"] else dict(out=out)


def _np_evict(case: dict, s: dict):
    b, kv, hd, keep, first, last = (case[x] for x in ("batch", "kv", "hd", "keep", "first", "last"))
    weights = s["weights_in"].double().cpu().numpy()
    got = dict(index=None, len=None, weights=np.zeros(s["weights_out"].shape))
    chosen = {}
    for i, n in enumerate(s["lens"].tolist()):
        for h in range(kv):
            left = np.arange(n)
            if n > keep:
                middle = left[first:n - last]
                best = middle[np.argsort(-weights[i, h, first:n - last], kind="stable")[:keep - first - last]]
                left = np.concatenate([left[:first], np.sort(best), left[n - last:]])
            chosen[i, h] = left
            got["weights"][i, h, :len(left)] = weights[i, h, left]
    for name, codes, scales in (("k", s["kc"], s["ks"]), ("v", s["vc"], s["vs"])):
        values, after = np.zeros((b, keep, kv, hd), np.float32), np.ones(s["to_ks"].shape)  # (every value is a float32)
        scales = scales.double().cpu().numpy()
        for (i, h), left in chosen.items():
            rows = codes[i, h, torch.from_numpy(left).to("cuda")].float().cpu().numpy()
            was = scales[i, h, left // BLOCK]
            for lo in range(0, len(left), BLOCK):
                scale = was[lo:lo + BLOCK].max()
                ratio = was[lo:lo + BLOCK] / scale
                moved = rows[lo:lo + BLOCK]
                if (ratio < 1).any():
                    moved = _np_round(moved * ratio[:, None], case["dtype"])
                values[i, lo:lo + len(moved), h] = moved * scale
                after[i, h, lo // BLOCK] = scale
        got[name], got[name + "_scale"] = values, after
    return {x: got[x] for x in ("index", "len", "weights", "k", "k_scale", "v", "v_scale")}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"append": _np_append, "attention": _f64_attention, "evict": _np_evict}[case["kind"]](case, s)
