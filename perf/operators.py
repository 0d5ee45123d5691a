"""Workloads of the paged-cache serving operators: appending rotated keys and
values to a paged KV cache, reading rows of it back, attention of one new token
per sequence over it, and token log probabilities.

Each case runs in two forms on the same inputs: the plain form (``own`` false),
elementary torch operations in float32, and the framework's operators (``own``
true). Head counts 32 / 4 with 64-wide heads, vocabulary 32000 and contexts up
to 2048 are this repository's model; the other sizes are generic.
"""

import importlib.util
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_FLOATS = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1}


def _package():
    if "lpta_b200" not in sys.modules:
        home = Path(__file__).resolve().parent.parent / "low-precision-transformer-accelerator-for-edge-llms_b200"
        spec = importlib.util.spec_from_file_location("lpta_b200", home / "__init__.py",
                                                      submodule_search_locations=[str(home)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["lpta_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["lpta_b200"]


# ----------------------------------------------------------------- the cases
def listed():
    return [
        # the one new token of an interactive session: launch latency
        {"name": "append-step-1", "op": "append", "mode": "step", "seqs": 1, "context": 700, "padded": 0,
         "heads": 32, "kv_heads": 4, "head_dim": 64, "page": 16, "in": "f32", "cache": "bf16"},
        # ragged prompts entering an INT8 cache from float32 activations, and the rows read back
        # (prefix attention over a stored prefix reads them in this way)
        {"name": "append-prompts-i8", "op": "append", "mode": "prompt", "seqs": 9, "context": 1500, "padded": 0,
         "heads": 32, "kv_heads": 4, "head_dim": 64, "page": 64, "in": "f32", "cache": "i8"},
        # a batch of full-length prompts, 16-bit activations and cache
        {"name": "append-prompts-bf16", "op": "append", "mode": "prompt", "seqs": 16, "context": 2048, "padded": 0,
         "heads": 32, "kv_heads": 4, "head_dim": 64, "page": 16, "in": "bf16", "cache": "bf16"},
        # one short prefix read back in full precision
        {"name": "read-prefix-i8", "op": "read", "seqs": 1, "context": 301, "kv_heads": 4, "head_dim": 64,
         "page": 16, "out": "f32", "cache": "i8"},
        # long contexts leaving the pool (moved to another worker): bandwidth
        {"name": "read-contexts-bf16", "op": "read", "seqs": 7, "context": 8192, "kv_heads": 8, "head_dim": 128,
         "page": 32, "out": "bf16", "cache": "bf16"},
        # the first step after a short prompt: latency
        {"name": "attend-1x17", "op": "attend", "seqs": 1, "context": 17, "padded": 0, "heads": 32, "kv_heads": 4,
         "head_dim": 64, "page": 16, "q": "bf16", "cache": "bf16"},
        # this repository's decode batch: 64 rows, three of them padding of a captured step,
        # contexts spread up to 2048, float32 activations over the INT8 cache
        {"name": "attend-64x2048-i8", "op": "attend", "seqs": 64, "context": 2048, "padded": 3, "heads": 32,
         "kv_heads": 4, "head_dim": 64, "page": 64, "q": "f32", "cache": "i8"},
        # a batch of longer contexts, five query heads a KV head, pages that are no power of two
        {"name": "attend-16x8192-f16", "op": "attend", "seqs": 16, "context": 8192, "padded": 0, "heads": 40,
         "kv_heads": 8, "head_dim": 128, "page": 48, "q": "f16", "cache": "f16"},
        # one very long context, ending inside a page: the work has to be split over its length
        {"name": "attend-1x131k-bf16", "op": "attend", "seqs": 1, "context": 131149, "padded": 0, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 128, "q": "bf16", "cache": "bf16"},
        # the answer's log probability with the alternatives of an API reply: latency
        {"name": "logprobs-1x32000", "op": "logprobs", "rows": 1, "vocab": 32000, "top_k": 20, "in": "f32"},
        # a decode batch, an odd vocabulary, 16-bit logits (many ties)
        {"name": "logprobs-64x50021-bf16", "op": "logprobs", "rows": 64, "vocab": 50021, "top_k": 5, "in": "bf16"},
        # scoring a whole prompt
        {"name": "logprobs-2048x32000", "op": "logprobs", "rows": 2048, "vocab": 32000, "top_k": 5, "in": "f32"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "logprobs"])
    if op == "logprobs":
        vocab = _log_int(rng, 500, 131072)
        rows = _log_int(rng, 1, max(1, min(4096, 64_000_000 // vocab)))
        return {"op": op, "rows": rows, "vocab": vocab, "top_k": rng.choice([0, 1, 5, 20, rng.randint(2, 32)]),
                "in": rng.choice(["f32", "bf16", "f16"])}
    head_dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 3, 4, 7, 8, 16])
    page = rng.choice([8, 16, 16, 32, 48, 64, 100, 128])
    cache = rng.choice(["i8", "bf16", "f16"])
    act = rng.choice(["f32", "bf16", "f16"])
    most = 100_000_000 // (kv_heads * head_dim * 4)  # cached rows of one case
    if op == "attend":
        seqs = _log_int(rng, 1, 256)
        context = _log_int(rng, 1, min(131072, 2 * most // (seqs + 1)))
        return {"op": op, "seqs": seqs, "context": context, "padded": rng.choice([0, 0, 1, 2]),
                "heads": kv_heads * group, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "q": act,
                "cache": cache}
    seqs = _log_int(rng, 1, 64)
    if op == "read":
        context = _log_int(rng, 1, min(16384, most // seqs))
        return {"op": op, "seqs": seqs, "context": context, "kv_heads": kv_heads, "head_dim": head_dim,
                "page": page, "out": act, "cache": cache}
    mode = rng.choice(["step", "prompt"])
    context = _log_int(rng, 1, min(4096, most // seqs if mode == "step" else most // (4 * seqs * max(1, group // 2))))
    return {"op": op, "mode": mode, "seqs": seqs, "context": context,
            "padded": rng.choice([0, 1]) if mode == "step" else 0, "heads": kv_heads * group,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "in": act, "cache": cache}


def _lengths(case):
    """Context of each sequence: the first one's is the whole, the others are spread below it."""
    n, c = case["seqs"], case["context"]
    return [c] + [1 + int((r * 0.6180339887) % 1.0 * (c - 1)) for r in range(1, n)]


def work(case):
    if case["op"] == "logprobs":
        r, v, k = case["rows"], case["vocab"], case["top_k"]
        return {"bytes": r * v * _BYTES[case["in"]] + r * (12 + 8 * k), "flops": 6 * r * v}
    lens, kv, d = _lengths(case), case["kv_heads"], case["head_dim"]
    stored = kv * d * _BYTES[case["cache"]] * 2 + (8 * kv if case["cache"] == "i8" else 0)  # a position of K and V
    table = 4 * sum(-(-x // case["page"]) for x in lens)
    if case["op"] == "attend":
        row = case["heads"] * d * _BYTES[case["q"]] * 2 + case["heads"] * 4 + 8
        return {"bytes": sum(lens) * stored + table + (case["seqs"] + case["padded"]) * row,
                "flops": 4 * sum(lens) * case["heads"] * d}
    if case["op"] == "read":
        return {"bytes": sum(lens) * (stored + 2 * kv * d * _BYTES[case["out"]] + 8) + table, "flops": 2 * sum(lens) * kv * d}
    step = case["mode"] == "step"
    tokens = case["seqs"] if step else sum(lens)
    angles = len(set(lens)) if step else case["context"]  # distinct positions: d / 2 cosines and sines each
    act = _BYTES[case["in"]]
    per = (2 * case["heads"] + 2 * kv) * d * act + stored + 8
    if case["cache"] == "i8":
        per += stored + 2 * kv * d * 4  # the rows read back
    return {"bytes": tokens * per + angles * d * 4 + table, "flops": 3 * tokens * (case["heads"] + kv) * d}


# ------------------------------------------------------------------- inputs
def _paged(case, gen, filled):
    """A pool with pages in random order, its block table, and random contents where ``filled``."""
    lens, ps, kv, d = _lengths(case), case["page"], case["kv_heads"], case["head_dim"]
    need = [-(-x // ps) for x in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = torch.nonzero(torch.arange(max(need)).unsqueeze(0) < torch.tensor(need).unsqueeze(1), as_tuple=True)
    table = table.cuda()
    table[at[0].cuda(), at[1].cuda()] = order[: sum(need)]
    shape = (pages, kv, ps, d)
    s = {"table": table, "k_scale": None, "v_scale": None}
    for name in ("k", "v"):
        if case["cache"] == "i8":
            s[name] = torch.zeros(shape, dtype=torch.int8, device="cuda")
            s[name + "_scale"] = torch.zeros(shape[:3], dtype=torch.float32, device="cuda")
            if filled:
                s[name] = torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)
                s[name + "_scale"] = torch.rand(shape[:3], generator=gen, device="cuda") * 0.02 + 0.005
        elif filled:
            s[name] = torch.randn(shape, generator=gen, device="cuda", dtype=_FLOATS[case["cache"]])
        else:
            s[name] = torch.zeros(shape, dtype=_FLOATS[case["cache"]], device="cuda")
    if filled and case["cache"] != "i8":
        s["k"][..., 3] *= 4  # keys have channels that stand out
    return s


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "logprobs":
        dt = _FLOATS[case["in"]]
        logits = torch.randn((case["rows"], case["vocab"]), generator=gen, device="cuda", dtype=dt)
        logits *= 2.5
        # a few likely tokens stand out in each row; the given ones are among them or not
        likely = torch.randint(0, case["vocab"] // 4, (case["rows"], 4), generator=gen, device="cuda")
        likely += torch.arange(4, device="cuda") * (case["vocab"] // 4)
        logits.scatter_(1, likely, (torch.rand(likely.shape, generator=gen, device="cuda") * 9 + 6).to(dt))
        other = torch.randint(0, case["vocab"], (case["rows"],), generator=gen, device="cuda")
        some = torch.rand(case["rows"], generator=gen, device="cuda") < 0.7
        return {"op": "logprobs", "logits": logits, "tokens": torch.where(some, likely[:, 0], other).to(torch.int32),
                "top_k": case["top_k"]}
    lens, d = _lengths(case), case["head_dim"]
    s = _paged(case, gen, case["op"] != "append")
    if case["op"] == "attend":
        rows = case["seqs"] + case["padded"]
        s["lengths"] = _i32(lens + [0] * case["padded"])
        s["seq"] = _i32(list(range(case["seqs"])) + [-1] * case["padded"])
        s["q"] = torch.randn((rows, case["heads"], d), generator=gen, device="cuda", dtype=_FLOATS[case["q"]]) * 1.5
    else:
        if case["op"] == "append" and case["mode"] == "step":
            s["seq"] = _i32(list(range(case["seqs"])) + [-1] * case["padded"])
            s["pos"] = _i32([x - 1 for x in lens] + [0] * case["padded"])
        else:
            s["seq"] = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).to(torch.int32).cuda()
            s["pos"] = torch.cat([torch.arange(x) for x in lens]).to(torch.int32).cuda()
        if case["op"] == "append":
            h, kv = case["heads"], case["kv_heads"]
            # queries, keys and values are columns of one projection's output
            qkv = torch.randn((s["seq"].numel(), h + 2 * kv, d), generator=gen, device="cuda",
                              dtype=_FLOATS[case["in"]])
            s["new_q"], s["new_k"], s["new_v"] = qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:]
            inv = 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float32) / d)
            ang = torch.arange(case["context"], device="cuda", dtype=torch.float32).unsqueeze(1) * inv
            s["cos"], s["sin"] = (torch.cat([f(ang)] * 2, 1).contiguous() for f in (torch.cos, torch.sin))
        else:
            s["out"] = _FLOATS[case["out"]]
    s["op"], s["live"] = case["op"], s["seq"].numel() - case.get("padded", 0)
    if own:  # the handle that a program keeps beside its pool's tensors
        s["handle"] = _package().PagedKVCache.from_tensors(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s


# ----------------------------------------------------------------- one pass
def run(state):
    return _RUN[state["op"]][own](state)


def _own_append(s):
    c = s["handle"]
    q = c.append(s["new_k"], s["new_v"], s["table"], s["seq"], s["pos"], s["cos"], s["sin"], q=s["new_q"])
    if s["k_scale"] is None:
        return {"q": q, "k": s["k"], "v": s["v"]}
    k, v = c.read(s["table"], s["seq"], s["pos"], dtype=torch.float32)
    return {"q": q, "k": k, "v": v}


def _own_read(s):
    k, v = s["handle"].read(s["table"], s["seq"], s["pos"], dtype=s["out"])
    return {"k": k, "v": v}


def _own_attend(s):
    out, lse = s["handle"].attend(s["q"], s["table"], s["lengths"], seq=s["seq"], return_lse=True)
    return {"out": out, "lse": lse}


def _own_logprobs(s):
    r = _package().token_logprobs(s["logits"], s["tokens"], top_k=s["top_k"])
    return {"logprob": r.logprob, "entropy": r.entropy, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs}


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    return x * cos.unsqueeze(1) + turned * sin.unsqueeze(1)


def _int8(x):
    peak = x.abs().amax(-1)
    scale = torch.where(peak == 0, torch.ones_like(peak), peak / torch.full_like(peak, 127.0))
    return torch.clamp(torch.round(x / scale.unsqueeze(-1)), -127, 127).to(torch.int8), scale


def _place(s, page_size):
    live = s["seq"] >= 0
    seq, pos = s["seq"].long().clamp_min(0), s["pos"].long()
    return live, s["table"][seq, pos // page_size].long(), pos % page_size


def _plain_append(s):
    pos = s["pos"].long()
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = _rotate(s["new_q"].float(), cos, sin).to(s["new_q"].dtype)
    k, v = _rotate(s["new_k"].float(), cos, sin), s["new_v"].float()
    _, page, off = _place(s, s["k"].shape[2])
    n = s["live"]  # padding comes last
    page, off, k, v = page[:n], off[:n], k[:n], v[:n]
    for name, x in (("k", k), ("v", v)):
        if s["k_scale"] is None:
            s[name][page, :, off] = x.to(s[name].dtype)
        else:
            s[name][page, :, off], s[name + "_scale"][page, :, off] = _int8(x)
    if s["k_scale"] is None:
        return {"q": q, "k": s["k"], "v": s["v"]}
    return {"q": q, **_plain_read({**s, "out": torch.float32})}


def _plain_read(s):
    live, page, off = _place(s, s["k"].shape[2])
    got = {}
    for name in ("k", "v"):
        x = s[name][page, :, off].float()
        if s["k_scale"] is not None:
            x = x * s[name + "_scale"][page, :, off].unsqueeze(-1)
        got[name] = (x * live.view(-1, 1, 1)).to(s["out"])
    return got


def _plain_attend(s):
    rows, heads, d = s["q"].shape
    pages = s["table"][s["seq"].long().clamp_min(0)].long()
    kv, ps = s["k"].shape[1:3]

    def gathered(name):  # [rows, kv heads, positions, d]
        x = s[name][pages].float()
        if s["k_scale"] is not None:
            x = x * s[name + "_scale"][pages].unsqueeze(-1)
        return x.transpose(1, 2).reshape(rows, kv, -1, d)

    q = s["q"].float().view(rows, kv, heads // kv, d)
    score = q @ gathered("k").transpose(-1, -2) * d ** -0.5
    hidden = torch.arange(score.shape[-1], device="cuda") >= s["lengths"].view(-1, 1, 1, 1)
    score = score.masked_fill(hidden, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = (p @ gathered("v")) / torch.where(total == 0, torch.ones_like(total), total)
    return {"out": out.view(rows, heads, d).to(s["q"].dtype), "lse": (top + torch.log(total)).view(rows, heads)}


def _plain_logprobs(s):
    x, vocab = s["logits"].float(), s["logits"].shape[1]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(1)
    entropy = torch.log(total).squeeze(1) - (e * (x - top)).sum(1) / total.squeeze(1)
    logprob = x.gather(1, s["tokens"].long().unsqueeze(1)).squeeze(1) - lse
    # the order of float32 as whole numbers above the index's complement: equal values go to the lowest index
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32)
    key = key + (vocab - 1 - torch.arange(vocab, device="cuda"))
    ids = vocab - 1 - (torch.topk(key, s["top_k"], dim=1).values & 0xFFFFFFFF)
    return {"logprob": logprob, "entropy": entropy, "top_ids": ids.to(torch.int32),
            "top_logprobs": x.gather(1, ids) - lse.unsqueeze(1)}


_RUN = {"append": (_plain_append, _own_append), "read": (_plain_read, _own_read),
        "attend": (_plain_attend, _own_attend), "logprobs": (_plain_logprobs, _own_logprobs)}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The operators' definitions in float64, sequence by sequence."""
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        # log p_i = x_i - log sum exp x,  H = -sum p log p
        logp = torch.log_softmax(s["logits"].double(), 1)
        return {"logprob": logp[torch.arange(case["rows"], device="cuda"), s["tokens"].long()],
                "entropy": torch.special.entr(logp.exp()).sum(1), "top_ids": None,
                "top_logprobs": logp.topk(case["top_k"], dim=1).values}
    lens, ps, d = _lengths(case), case["page"], case["head_dim"]
    table = s["table"].cpu().numpy()

    def sequence(i, n, name):  # the n first rows of sequence i: [kv heads, n, d]
        pages = torch.from_numpy(table[i, : -(-n // ps)].astype(np.int64)).cuda()
        x = s[name][pages].double()
        if case["cache"] == "i8":
            x = x * s[name + "_scale"][pages].double().unsqueeze(-1)
        return x.permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, d)[:, :n]

    if case["op"] == "read":
        return {name: torch.cat([sequence(i, n, name).transpose(0, 1) for i, n in enumerate(lens)])
                for name in ("k", "v")}
    if case["op"] == "attend":
        rows, heads = case["seqs"] + case["padded"], case["heads"]
        out = torch.zeros((rows, heads, d), dtype=torch.float64, device="cuda")
        lse = torch.full((rows, heads), -math.inf, dtype=torch.float64, device="cuda")
        for i, n in enumerate(lens):
            q = s["q"][i].double().view(case["kv_heads"], -1, d)
            score = torch.einsum("hgd,hnd->hgn", q, sequence(i, n, "k")) / math.sqrt(d)
            lse[i] = torch.logsumexp(score, -1).flatten()
            out[i] = torch.einsum("hgn,hnd->hgd", torch.softmax(score, -1), sequence(i, n, "v")).reshape(heads, d)
        return {"out": out, "lse": lse}
    # append: pairs (x_j, x_{j + d/2}) turn by the position's angle
    at, half = s["pos"].long(), d // 2
    c, w = (s[t].double()[at][:, None, :half] for t in ("cos", "sin"))

    def turned(x):
        a, b = x.double()[..., :half], x.double()[..., half:]
        return torch.cat([a * c - b * w, b * c + a * w], -1)

    got = {"q": turned(s["new_q"])}
    seq, pos = s["seq"].cpu().numpy(), s["pos"].cpu().numpy()
    live = np.nonzero(seq >= 0)[0]
    page = torch.from_numpy(table[seq[live], pos[live] // ps].astype(np.int64)).cuda()
    off = torch.from_numpy((pos[live] % ps).astype(np.int64)).cuda()
    for name, x in (("k", turned(s["new_k"])), ("v", s["new_v"].double())):
        if case["cache"] == "i8":
            step = x.abs().amax(-1, keepdim=True) / 127
            step[step == 0] = 1
            got[name] = torch.clamp(torch.round(x / step), -127, 127) * step
            got[name][torch.from_numpy(seq < 0).cuda()] = 0
        else:
            whole = s[name].double()
            whole[page, :, off] = x[torch.from_numpy(live).cuda()]
            got[name] = whole
    return got
