"""Attention and its key-value cache, as cases to be timed.

  prompt  ``packed_attention``: attention within packed sequences of different
          lengths, grouped heads, causal or not; forward alone as in serving
          (q, k and v views of one projection; a chunk of a prompt over all of
          its keys where the keys outnumber the queries), or with all gradients
  decode  ``paged_attention``: one new token a sequence over its pages of a
          key-value cache, in bf16 or in E4M3 with a power of two a row
  cache   ``append_kv`` and ``read_kv``: new tokens written into the pages of
          their sequences, quantised where the cache is, and whole sequences
          read back, as a chunk of a prompt needs them

``own`` False computes them from elementary torch operations in 32 bits,
rounded once; ``own`` True through the package's entry points.
"""

import importlib
import math
import random

import torch

own = False

DEVICE = "cuda"


def listed():
    return [
        # one short question, served: the smallest prompt
        {"name": "prompt 333 h16/2 d128", "kind": "prompt", "tokens": 333, "keys": 333, "seqs": 1, "heads": 16,
         "kv_heads": 2, "dim": 128, "causal": True, "train": False, "mix": 0},
        # a prefill batch of 11 prompts of different lengths
        {"name": "prompt packed 8192 h32/8 d128", "kind": "prompt", "tokens": 8192, "keys": 8192, "seqs": 11,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "train": False, "mix": 1},
        # one long document, few heads a GPU
        {"name": "prompt 16384 h8/1 d128", "kind": "prompt", "tokens": 16384, "keys": 16384, "seqs": 1, "heads": 8,
         "kv_heads": 1, "dim": 128, "causal": True, "train": False, "mix": 0},
        # the next chunks of two prompts, over all keys so far
        {"name": "prompt chunk 1000/16000 h32/4 d128", "kind": "prompt", "tokens": 1000, "keys": 16000, "seqs": 2,
         "heads": 32, "kv_heads": 4, "dim": 128, "causal": True, "train": False, "mix": 2},
        # a small ragged training batch, narrow heads, seen both ways
        {"name": "prompt train 777 h12/4 d64", "kind": "prompt", "tokens": 777, "keys": 777, "seqs": 5, "heads": 12,
         "kv_heads": 4, "dim": 64, "causal": False, "train": True, "mix": 3},
        # a training batch of 8,192 tokens in three documents: the largest call
        {"name": "prompt train 8192 h32/8 d128", "kind": "prompt", "tokens": 8192, "keys": 8192, "seqs": 3,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "train": True, "mix": 4},
        # one short conversation: the smallest call
        {"name": "decode 1x200 h32/8 d128", "kind": "decode", "longest": 200, "seqs": 1, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "cache": "bf16", "idle": False, "mix": 0},
        # 16 ragged conversations over a quantised cache, one slot of the batch idle
        {"name": "decode 16x4000 h64/8 d128 e4m3", "kind": "decode", "longest": 4000, "seqs": 16, "heads": 64,
         "kv_heads": 8, "dim": 128, "page": 64, "cache": "e4m3", "idle": True, "mix": 1},
        # one very long document
        {"name": "decode 1x131000 h32/4 d128", "kind": "decode", "longest": 131000, "seqs": 1, "heads": 32,
         "kv_heads": 4, "dim": 128, "page": 16, "cache": "bf16", "idle": False, "mix": 0},
        # a full serving batch
        {"name": "decode 64x8192 h32/8 d128 e4m3", "kind": "decode", "longest": 8192, "seqs": 64, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "cache": "e4m3", "idle": False, "mix": 2},
        # the second turn of one short conversation
        {"name": "cache 100+37 h4 d128", "kind": "cache", "before": 100, "tokens": 37, "seqs": 1, "kv_heads": 4,
         "dim": 128, "page": 16, "cache": "bf16", "mix": 0},
        # chunks of 8 prompts into a quantised cache, and all that the 8 have so far
        {"name": "cache 30000+4096 h8 d128 e4m3", "kind": "cache", "before": 30000, "tokens": 4096, "seqs": 8,
         "kv_heads": 8, "dim": 128, "page": 64, "cache": "e4m3", "mix": 5},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "decode", "decode", "cache"])
    kv_heads = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    case = {"kind": kind, "kv_heads": kv_heads, "dim": dim, "mix": rng.randrange(1000)}
    if kind == "prompt":
        case["heads"] = kv_heads * rng.choice([1, 2, 4, 5, 8])
        case["train"] = rng.random() < 0.5
        tokens = _log_uniform(rng, 16, 16384)
        tokens = min(tokens, int(8192 * math.sqrt(32 * 128 / (case["heads"] * max(dim, 128)))))
        chunk = not case["train"] and rng.random() < 0.3
        case.update(tokens=max(1, tokens // rng.choice([3, 9, 27])) if chunk else tokens, keys=tokens,
                    seqs=min(1 if chunk else tokens, rng.choice([1, 2, 7, 30])), causal=chunk or rng.random() < 0.8)
        return case
    case.update(page=rng.choice([16, 32, 64, 128]), cache=rng.choice(["bf16", "e4m3"]))
    if kind == "decode":
        case["heads"] = kv_heads * rng.choice([1, 3, 4, 8, 12])
        case["seqs"] = _log_uniform(rng, 1, 128)
        case["longest"] = max(1, min(_log_uniform(rng, 16, 131072), 64 * 8192 * 8 * 128 // (case["seqs"] * kv_heads * dim)))
        case["idle"] = case["seqs"] > 1 and rng.random() < 0.3
        return case
    case.update(seqs=rng.choice([1, 3, 8]), before=_log_uniform(rng, 16, 60000), tokens=_log_uniform(rng, 8, 8192))
    return case


# ------------------------------------------------------------------ inputs --


def _shares(total, seqs, mix, least=1):
    """`total` in `seqs` parts of different sizes, each `least` or more."""
    rng = random.Random(mix)
    weights = [0.2 + rng.random() for _ in range(seqs)]
    free, parts = total - seqs * least, []
    for i, w in enumerate(weights):
        parts.append(least + int(free * w / sum(weights)))
    parts[-1] += total - sum(parts)
    return parts


def _lengths(case):
    """(queries, keys) of each sequence of a prompt; keys of each of a decode
    step; (before, new) of each of a cache's."""
    seqs, mix = case["seqs"], case["mix"]
    if case["kind"] == "prompt":
        queries = _shares(case["tokens"], seqs, mix)
        if case["keys"] == case["tokens"]:
            return queries, queries
        before = _shares(case["keys"] - case["tokens"], seqs, mix + 1, 0)
        return queries, [q + b for q, b in zip(queries, before)]
    if case["kind"] == "decode":
        rng = random.Random(mix)
        lengths = [case["longest"]] + [1 + int((case["longest"] - 1) * rng.random() ** 0.5) for _ in range(seqs - 1)]
        if case["idle"]:
            lengths[-1] = 0
        return lengths
    return _shares(case["before"], seqs, mix, 0), _shares(case["tokens"], seqs, mix + 1, 0)


def _offsets(lengths):
    got = [0]
    for n in lengths:
        got.append(got[-1] + n)
    return torch.tensor(got, dtype=torch.int32, device=DEVICE)


class _Inputs:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE)
        self.g.manual_seed(int(seed))

    def normal(self, *shape, std=1.0):
        return torch.randn(shape, generator=self.g, device=DEVICE, dtype=torch.float32).mul_(std)

    def keys(self, *shape):
        """Rows of keys: a few channels are larger than the others."""
        k = self.normal(*shape)
        k[..., :: shape[-1] // 4] *= 3
        return k

    def integers(self, high, *shape, dtype=torch.int32):
        return torch.randint(high, shape, generator=self.g, device=DEVICE, dtype=dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device=DEVICE, dtype=torch.int64)


def _pages(rng, case, lengths):
    """A cache whose pages hold `lengths` tokens of each sequence, in any
    order, and what was there before in the rest of them."""
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    need = [-(-n // page) for n in lengths]
    count = sum(need) + 3
    s = {"table": torch.full((len(lengths), max(1, max(need))), -1, dtype=torch.int32, device=DEVICE)}
    order, at = rng.order(count).to(torch.int32), 0
    for i, n in enumerate(need):
        s["table"][i, :n] = order[at:at + n]
        at += n
    for name, values in (("k", rng.keys), ("v", rng.normal)):
        if case["cache"] == "bf16":
            s[name + "_pages"] = values(count, heads, page, dim).to(torch.bfloat16)
            s[name + "_scales"] = None
        else:
            x = values(count, heads, page, dim)
            top = x.abs().amax(3, keepdim=True)
            step = torch.exp2(torch.ceil(torch.log2(top / 448)))
            s[name + "_pages"] = (x / step).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            s[name + "_scales"] = (torch.log2(step[..., 0]) + 127).to(torch.uint8)
    return s


def prepare(case, seed):
    rng, s = _Inputs(seed), {"case": case}
    heads, kv_heads, dim = case.get("heads"), case["kv_heads"], case["dim"]
    if case["kind"] == "prompt":
        queries, keys = _lengths(case)
        s["offsets"] = _offsets(queries)
        s["key_offsets"] = _offsets(keys) if keys != queries else None
        tokens, all_keys = case["tokens"], case["keys"]
        if case["train"]:
            s["q"] = rng.normal(tokens, heads, dim).to(torch.bfloat16).requires_grad_()
            s["k"] = rng.keys(all_keys, kv_heads, dim).to(torch.bfloat16).requires_grad_()
            s["v"] = rng.normal(all_keys, kv_heads, dim).to(torch.bfloat16).requires_grad_()
            s["d_out"] = rng.normal(tokens, heads, dim, std=0.1).to(torch.bfloat16)
        elif tokens == all_keys:  # views of one projection's output
            joined = rng.normal(tokens, heads + 2 * kv_heads, dim).to(torch.bfloat16)
            s["q"], s["k"], s["v"] = joined.split([heads, kv_heads, kv_heads], 1)
            s["k"][..., :: dim // 4] *= 3
        else:
            s["q"] = rng.normal(tokens, heads, dim).to(torch.bfloat16)
            s["k"] = rng.keys(all_keys, kv_heads, dim).to(torch.bfloat16)
            s["v"] = rng.normal(all_keys, kv_heads, dim).to(torch.bfloat16)
    elif case["kind"] == "decode":
        lengths = _lengths(case)
        s.update(_pages(rng, case, lengths))
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
        s["q"] = rng.normal(case["seqs"], heads, dim).to(torch.bfloat16)
    else:
        before, new = _lengths(case)
        after = [b + n for b, n in zip(before, new)]
        s.update(_pages(rng, case, after))
        s["before"] = torch.tensor(before, dtype=torch.int32, device=DEVICE)
        s["offsets"], s["key_offsets"] = _offsets(new), _offsets(after)
        s["k"] = rng.keys(case["tokens"], kv_heads, dim).to(torch.bfloat16)
        s["v"] = rng.normal(case["tokens"], kv_heads, dim).to(torch.bfloat16)
    return s


# --------------------------------------------------------------------- run --


def _package():
    return importlib.import_module("glm53-flash-mlx_amd")


def _attend(q, k, v, seen):
    """q [..., n, dim], k and v [..., m, dim], seen [..., n, m]: softmax over
    the keys that are seen, 0 where there is none."""
    s = (q @ k.transpose(-1, -2)) / math.sqrt(q.shape[-1])
    s = s.masked_fill(~seen, -math.inf)
    top = s.detach().amax(-1, keepdim=True)
    p = torch.exp(s - top.masked_fill(top == -math.inf, 0))
    total = p.sum(-1, keepdim=True)
    return (p / total.masked_fill(total == 0, 1)) @ v


def _numbers(offsets, count):
    """The sequence of each of `count` rows, and its place in it."""
    rows = torch.arange(count, device=DEVICE)
    seq = torch.searchsorted(offsets.long(), rows, right=True) - 1
    return seq, rows - offsets.long()[seq]


def _seen(s, tokens, keys):
    offsets = s["offsets"]
    key_offsets = s["key_offsets"] if s["key_offsets"] is not None else offsets
    (qs, qi), (ks, ki) = _numbers(offsets, tokens), _numbers(key_offsets, keys)
    seen = qs[:, None] == ks[None, :]
    if s["case"]["causal"]:
        more = key_offsets.diff().long() - offsets.diff().long()
        seen = seen & (ki[None, :] <= (qi + more[qs])[:, None])
    return seen


def _plain_prompt(s):
    case = s["case"]
    group = case["heads"] // case["kv_heads"]
    q, k, v = (s[n].float().transpose(0, 1) for n in ("q", "k", "v"))
    q = q.reshape(case["kv_heads"], group, case["tokens"], case["dim"])
    out = _attend(q, k[:, None], v[:, None], _seen(s, case["tokens"], case["keys"]))
    return out.reshape(case["heads"], case["tokens"], case["dim"]).transpose(0, 1).contiguous().to(torch.bfloat16)


def _run_prompt(s):
    if own:
        out = _package().packed_attention(s["q"], s["k"], s["v"], s["offsets"], s["key_offsets"],
                                          causal=s["case"]["causal"])
    else:
        out = _plain_prompt(s)
    got = {"out": out}
    if s["case"]["train"]:
        grads = torch.autograd.grad([out], [s["q"], s["k"], s["v"]], [s["d_out"]])
        got.update(d_q=grads[0], d_k=grads[1], d_v=grads[2])
    return got


def _power(e):
    """2^e in 32 bits, exactly: its exponent's bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _values(pages, scales):
    if scales is None:
        return pages.float()
    return pages.view(torch.float8_e4m3fn).float() * _power(scales.to(torch.int32) - 127)[..., None]


def _gather(s, name):
    """All positions of every sequence, in 32 bits: [seqs, kv_heads, positions, dim]."""
    case, table = s["case"], s["table"].clamp(min=0).long()
    scales = s[name + "_scales"]
    x = _values(s[name + "_pages"][table], None if scales is None else scales[table])  # [seqs, pages, heads, page, dim]
    return x.transpose(1, 2).reshape(table.shape[0], case["kv_heads"], -1, case["dim"])


def _run_decode(s):
    if own:
        return _package().paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"],
                                          k_scales=s["k_scales"], v_scales=s["v_scales"])
    case, k, v = s["case"], _gather(s, "k"), _gather(s, "v")
    seen = torch.arange(k.shape[2], device=DEVICE)[None, :] < s["lengths"].long()[:, None]
    v = v.masked_fill(~seen[:, None, :, None], 0)  # whatever lies behind a sequence's last token
    q = s["q"].float().view(case["seqs"], case["kv_heads"], -1, case["dim"])
    return _attend(q, k, v, seen[:, None, None, :]).reshape(case["seqs"], case["heads"], -1).to(torch.bfloat16)


def _plain_append(s, name):
    """New rows into their pages: as they are, or as E4M3 codes of the row
    divided by the smallest power of two that brings it to 448 or less."""
    case, x = s["case"], s[name]
    seq, place = _numbers(s["offsets"], case["tokens"])
    position = s["before"].long()[seq] + place
    page, slot = s["table"][seq, position // case["page"]].long(), position % case["page"]
    if s[name + "_scales"] is None:
        s[name + "_pages"][page, :, slot] = x
        return
    x = x.float()
    part, power = torch.frexp(x.abs().amax(2))  # part in [0.5, 1)
    power = (power - 9 + (part > 0.875)).clamp(min=-117).masked_fill(part == 0, -117)
    codes = (x * _power(-power)[..., None]).to(torch.float8_e4m3fn)
    s[name + "_pages"][page, :, slot] = codes.view(torch.uint8)
    s[name + "_scales"][page, :, slot] = (power + 127).to(torch.uint8)


def _plain_read(s, name, total):
    case = s["case"]
    seq, position = _numbers(s["key_offsets"], total)
    page, slot = s["table"][seq, position // case["page"]].long(), position % case["page"]
    scales = s[name + "_scales"]
    x = _values(s[name + "_pages"][page, :, slot], None if scales is None else scales[page, :, slot])
    return x.to(torch.bfloat16)


def _run_cache(s):
    total = s["case"]["before"] + s["case"]["tokens"]
    if own:
        package = _package()
        package.append_kv(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["before"], s["offsets"],
                          k_scales=s["k_scales"], v_scales=s["v_scales"])
        k, v = package.read_kv(s["k_pages"], s["v_pages"], s["table"], s["key_offsets"], total,
                               k_scales=s["k_scales"], v_scales=s["v_scales"])
        return {"k": k, "v": v}
    for name in ("k", "v"):
        _plain_append(s, name)
    return {name: _plain_read(s, name, total) for name in ("k", "v")}


def run(state):
    return {"prompt": _run_prompt, "decode": _run_decode, "cache": _run_cache}[state["case"]["kind"]](state)


# -------------------------------------------------------------------- work --


def _pairs(queries, keys, causal):
    """Pairs of a query and a key that it sees."""
    if not causal:
        return queries * keys
    first = keys - queries + 1  # keys that the first query sees
    return queries * (first + keys) // 2


def work(case):
    heads, kv_heads, dim = case.get("heads", 0), case["kv_heads"], case["dim"]
    if case["kind"] == "prompt":
        pairs = sum(_pairs(q, k, case["causal"]) for q, k in zip(*_lengths(case)))
        total, flops = 2 * dim * (2 * case["tokens"] * heads + 2 * case["keys"] * kv_heads), 4 * pairs * heads * dim
        if case["train"]:  # d_out, d_q, d_k, d_v; five products for two
            total, flops = total + 2 * dim * (2 * case["tokens"] * heads + 2 * case["keys"] * kv_heads), 3.5 * flops
        return {"bytes": total, "flops": flops}
    row = kv_heads * (2 * dim if case["cache"] == "bf16" else dim + 1)
    if case["kind"] == "decode":
        tokens = sum(_lengths(case))
        return {"bytes": 2 * tokens * row + 4 * case["seqs"] * heads * dim, "flops": 4 * tokens * heads * dim}
    new, after = case["tokens"], case["before"] + case["tokens"]
    return {"bytes": 2 * (new + after) * (row + 2 * kv_heads * dim), "flops": 2 * (new + after) * kv_heads * dim}


# ------------------------------------------------------------------- exact --


def _exact_head(q, k, v, seen, d_out=None):
    """One head of one sequence in 64 bits, with its gradients."""
    scale = q.shape[1] ** -0.5
    weights = torch.where(seen, scale * q.matmul(k.t()), -math.inf).softmax(1).nan_to_num(0.0)
    out = weights.matmul(v)
    if d_out is None:
        return out, None, None, None
    d_weights = d_out.matmul(v.t())
    d_scores = weights * (d_weights - (weights * d_weights).sum(1, keepdim=True))
    return out, scale * d_scores.matmul(k), scale * d_scores.t().matmul(q), weights.t().matmul(d_out)


def _exact_prompt(s):
    case = s["case"]
    group = case["heads"] // case["kv_heads"]
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    got = {"out": torch.zeros_like(q)}
    if case["train"]:
        got.update(d_q=torch.zeros_like(q), d_k=torch.zeros_like(k), d_v=torch.zeros_like(v))
    a = b = 0
    for n, m in zip(*_lengths(case)):
        seen = torch.ones(n, m, dtype=torch.bool, device=DEVICE)
        if case["causal"]:
            seen = seen.tril(m - n)
        rows, cols = slice(a, a + n), slice(b, b + m)
        for h in range(case["heads"]):
            j = h // group
            d_out = s["d_out"][rows, h].double() if case["train"] else None
            out, d_q, d_k, d_v = _exact_head(q[rows, h], k[cols, j], v[cols, j], seen, d_out)
            got["out"][rows, h] = out
            if case["train"]:
                got["d_q"][rows, h] = d_q
                got["d_k"][cols, j] += d_k
                got["d_v"][cols, j] += d_v
        a, b = a + n, b + m
    return got


def _exact_pages(s, name, i, length):
    """Sequence i's first `length` rows in 64 bits, [length, kv_heads, dim]."""
    case = s["case"]
    pages = s["table"][i, : -(-length // case["page"])].long()
    x = s[name + "_pages"].index_select(0, pages)
    if s[name + "_scales"] is None:
        x = x.double()
    else:
        power = s[name + "_scales"].index_select(0, pages).long() - 127
        x = x.view(torch.float8_e4m3fn).double() * (power + 1023 << 52).view(torch.float64).unsqueeze(3)
    return x.permute(0, 2, 1, 3).reshape(-1, case["kv_heads"], case["dim"])[:length]


def _exact_decode(s):
    case, q = s["case"], s["q"].double()
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros_like(q)
    for i, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        k, v = _exact_pages(s, "k", i, n), _exact_pages(s, "v", i, n)
        seen = torch.ones(group, n, dtype=torch.bool, device=DEVICE)
        for j in range(case["kv_heads"]):
            rows = slice(j * group, (j + 1) * group)
            out[i, rows] = _exact_head(q[i, rows], k[:, j], v[:, j], seen)[0]
    return out


def _exact_stored(x, cache):
    """What a cache holds of rows x."""
    x = x.double()
    if cache == "bf16":
        return x
    top = x.abs().amax(2, keepdim=True)
    step = torch.full_like(top, 2.0**-117)
    for _ in range(250):  # the smallest power of two that brings the row to 448 or less
        step = torch.where(top > 448 * step, 2 * step, step)
    y = x / step
    spacing = (torch.frexp(y.abs().clamp(min=2.0**-6))[1].long() - 4 + 1023 << 52).view(torch.float64)
    return torch.round(y / spacing) * spacing * step


def _exact_cache(s):
    case, got = s["case"], {}
    before, new = _lengths(case)
    for name in ("k", "v"):
        rows, at = [], 0
        stored = _exact_stored(s[name], case["cache"])
        for i, (b, n) in enumerate(zip(before, new)):
            rows += [_exact_pages(s, name, i, b), stored[at:at + n]]
            at += n
        got[name] = torch.cat(rows)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"prompt": _exact_prompt, "decode": _exact_decode, "cache": _exact_cache}[case["kind"]](s)
