"""Timed cases of the attention operators: packed prompts (forward, and forward
with backward), appending to a paged cache with the position rotation, and
attention of new tokens over that cache.

Every operator has a plain form here, written in elementary tensor operations
in 32 bits, and a call of the framework's own kernels (`own`).  `exact` gives
the same results from the definition in 64 bits.

Layouts: q [rows][heads][dim], k and v [rows][kv_heads][dim], sequences packed
along the rows as (offset, length) pairs; a cache is [pages][kv_heads]
[page_size][dim], and row s of the page table lists the pages of sequence s.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # One new token for each of 32 running sequences: the step between two tokens of a
        # serving loop, where the latency of a launch is what a user sees.
        {"name": "append_decode", "kind": "append", "type": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "rot": 128, "interleaved": False, "page": 16, "seqs": 32, "new_max": 1,
         "past_max": 2048, "lens": 1},
        # The tokens of a batch of ragged prompts go into the cache; partial rotation, pairs
        # next to each other.
        {"name": "append_prompts", "kind": "append", "type": "f16", "heads": 32, "kv_heads": 8,
         "dim": 128, "rot": 64, "interleaved": True, "page": 64, "seqs": 24, "new_max": 2048,
         "past_max": 512, "lens": 2},
        # The smallest serving call: four short conversations, one token each.
        {"name": "decode_small", "kind": "paged", "type": "f16", "heads": 16, "kv_heads": 4,
         "dim": 64, "page": 16, "seqs": 4, "new_max": 1, "past_max": 500, "lens": 3},
        # A full serving batch of ragged contexts, one token each.
        {"name": "decode_batch", "kind": "paged", "type": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "seqs": 64, "new_max": 1, "past_max": 8192, "lens": 4},
        # One sequence with a very long context: few rows, a long axis.
        {"name": "decode_long", "kind": "paged", "type": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 32, "seqs": 1, "new_max": 1, "past_max": 131072, "lens": 5},
        # Chunked prefill: pieces of prompts behind cached contexts.
        {"name": "chunk_prefill", "kind": "paged", "type": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "seqs": 6, "new_max": 1024, "past_max": 8192, "lens": 6},
        # A few tokens at a time (checking drafted tokens), group of three heads, narrow heads.
        {"name": "chunk_few", "kind": "paged", "type": "f16", "heads": 24, "kv_heads": 8,
         "dim": 64, "page": 16, "seqs": 17, "new_max": 9, "past_max": 3000, "lens": 7},
        # Whole prompts of very different lengths, packed, causal, grouped heads.
        {"name": "prompts", "kind": "prompt", "type": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "causal": True, "seqs": 9, "len_max": 8192, "lens": 8},
        # Short ragged prompts with narrow heads, odd lengths down to one token.
        {"name": "prompts_short", "kind": "prompt", "type": "f16", "heads": 12, "kv_heads": 12,
         "dim": 64, "causal": True, "seqs": 40, "len_max": 333, "lens": 9},
        # A training step's attention: one packed row of documents, forward and backward.
        {"name": "train_packed", "kind": "train", "type": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "causal": True, "seqs": 5, "len_max": 4096, "lens": 10},
        # An encoder's training step: no causal mask, as many key heads as query heads.
        {"name": "train_encoder", "kind": "train", "type": "f16", "heads": 16, "kv_heads": 16,
         "dim": 64, "causal": False, "seqs": 30, "len_max": 512, "lens": 11},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "paged", "paged", "prompt", "train"])
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    case = {"kind": kind, "type": rng.choice(["bf16", "f16"]), "heads": kv_heads * group,
            "kv_heads": kv_heads, "dim": rng.choice([64, 64, 128, 128, 80, 96]),
            "lens": rng.randrange(1 << 30)}
    if case["heads"] > 32:
        case["heads"] = kv_heads
    if kind in ("append", "paged"):
        case["page"] = rng.choice([1, 8, 16, 32, 64, 128])
        if kind == "append" or rng.random() < 0.4:
            case["seqs"] = _log_uniform(rng, 1, 32)
            case["new_max"] = _log_uniform(rng, 1, 1024)
            case["past_max"] = _log_uniform(rng, 1, 4096)
        else:
            case["seqs"] = _log_uniform(rng, 1, 64)
            case["new_max"] = 1
            case["past_max"] = _log_uniform(rng, 1, 16384)
        if kind == "append":
            case["rot"] = 2 * rng.randint(1, case["dim"] // 2)
            case["interleaved"] = rng.random() < 0.5
    else:
        case["causal"] = rng.random() < 0.8
        case["seqs"] = _log_uniform(rng, 1, 40)
        top = 4096 if kind == "prompt" else 2048
        case["len_max"] = _log_uniform(rng, 1, top if case["seqs"] < 8 else top // 4)
    return case


def _ragged(rng, n, top):
    """n lengths in 1..top: one of them `top`, the others spread over its logarithm."""
    lens = [_log_uniform(rng, max(1, top // 64), top) for _ in range(n)]
    lens[rng.randrange(n)] = top
    return lens


def _lengths(case):
    """(new tokens, cached tokens) of every sequence; a case fixes them, seeds do not."""
    rng = random.Random(case["lens"])
    if case["kind"] in ("append", "paged"):
        return _ragged(rng, case["seqs"], case["new_max"]), _ragged(rng, case["seqs"], case["past_max"])
    return _ragged(rng, case["seqs"], case["len_max"]), [0] * case["seqs"]


def _pairs(case):
    """Visible (query, key) pairs of one head."""
    new, past = _lengths(case)
    if case["kind"] == "paged" or case.get("causal"):
        return sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    return sum(n * n for n in new)


def work(case):
    new, past = _lengths(case)
    rows, h, hk, d = sum(new), case["heads"], case["kv_heads"], case["dim"]
    q, kv = 2 * rows * h * d, 2 * rows * hk * d
    if case["kind"] == "append":
        return {"bytes": 2 * (q + 2 * kv), "flops": 3 * rows * (h + hk) * case["rot"]}
    if case["kind"] == "paged":
        keys = sum(n + p for n, p in zip(new, past))
        return {"bytes": 2 * q + 2 * 2 * keys * hk * d, "flops": 4 * d * h * _pairs(case)}
    if case["kind"] == "prompt":
        return {"bytes": 2 * q + 2 * kv + 4 * rows * h, "flops": 4 * d * h * _pairs(case)}
    # forward (4) and backward (10): q, k, v, dout in; out and three gradients back
    return {"bytes": 4 * q + 4 * kv, "flops": 14 * d * h * _pairs(case)}


# ------------------------------------------------------------------- the inputs
def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        _prepare_own(st)
    return st


def _inputs(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    t = DTYPES[case["type"]]
    new, past = _lengths(case)
    rows, h, hk, d = sum(new), case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(t)

    offsets = [0]
    for n in new[:-1]:
        offsets.append(offsets[-1] + n)
    st = {"case": case, "new": new, "past": past, "first": offsets, "rows": rows,
          "scale": 1.0 / math.sqrt(d),
          "offsets": torch.tensor(offsets, dtype=torch.int64, device=dev),
          "lens": torch.tensor(new, dtype=torch.int64, device=dev),
          "q": normal(rows, h, d)}
    if case["kind"] in ("append", "paged"):
        page = case["page"]
        need = [-(-(n + p) // page) for n, p in zip(new, past)]
        cols, total = max(need), sum(need)
        order = torch.randperm(total, generator=gen, device=dev).tolist()
        table = np.zeros((len(new), cols), np.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        st.update(table=torch.from_numpy(table).to(dev), cols=cols, pages=total,
                  past_lens=torch.tensor(past, dtype=torch.int64, device=dev),
                  k_pages=normal(total, hk, page, d), v_pages=normal(total, hk, page, d))
    if case["kind"] != "paged":
        st["k"], st["v"] = normal(rows, hk, d), normal(rows, hk, d)
    if case["kind"] == "append":
        half = case["rot"] // 2
        st["freqs"] = torch.tensor([10000.0 ** (-i / half) for i in range(half)],
                                   dtype=torch.float32, device=dev)
    if case["kind"] == "train":
        st["dout"] = normal(rows, h, d)
    return st


def _prepare_own(st):
    from futhark_amd import kernels
    case, dev = st["case"], "cuda"
    K = kernels.Kernels()
    st["K"], st["t"] = K, case["type"]
    st["failure"] = torch.zeros(1, dtype=torch.int32, device=dev)
    st["out"] = torch.zeros_like(st["q"])
    if case["kind"] == "paged":
        size = K.attention_paged_workspace_bytes(st["rows"], case["heads"], case["kv_heads"], case["dim"],
                                                 len(st["new"]), case["page"], st["cols"])
        st["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device=dev)
        st["workspace_bytes"] = size
    if case["kind"] in ("prompt", "train"):
        st["lse"] = torch.zeros(st["rows"], case["heads"], dtype=torch.float32, device=dev)
    if case["kind"] == "train":
        st["dq"], st["dk"], st["dv"] = (torch.zeros_like(st[x]) for x in "qkv")
        size = K.attention_grad_workspace_bytes(st["rows"], st["rows"], case["heads"], case["kv_heads"],
                                                case["dim"], len(st["new"]))
        st["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device=dev)
        st["workspace_bytes"] = size


# ------------------------------------------------------------- the plain forms
def _rotate(x, pos, freqs, rot, interleaved):
    angle = pos.double()[:, None] * freqs.double()[None, :]
    c, s = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    y = x.float().clone()
    if interleaved:
        a, b = y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = y[..., :rot // 2].clone(), y[..., rot // 2:rot].clone()
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return y.to(x.dtype)


def _plain_append(st):
    case, page = st["case"], st["case"]["page"]
    dev = st["q"].device
    pos = torch.cat([torch.arange(p, p + n, device=dev) for n, p in zip(st["new"], st["past"])])
    seq = torch.repeat_interleave(torch.arange(len(st["new"]), device=dev), st["lens"],
                                  output_size=st["rows"])
    slot, pages = pos % page, st["table"][seq, pos // page].long()
    st["k_pages"][pages, :, slot] = _rotate(st["k"], pos, st["freqs"], case["rot"], case["interleaved"])
    st["v_pages"][pages, :, slot] = st["v"]
    return [_rotate(st["q"], pos, st["freqs"], case["rot"], case["interleaved"]), st["k_pages"], st["v_pages"]]


def _scores(q, k, scale, behind):
    """q [heads][n][dim] on k [kv_heads][keys][dim] in 32 bits; `behind` cached keys before the
    first query for a causal mask, None without one."""
    g = q.shape[0] // k.shape[0]
    s = torch.matmul(q, k.repeat_interleave(g, 0).transpose(1, 2).contiguous()) * scale
    if behind is not None:
        n, keys = s.shape[1:]
        see = torch.arange(keys, device=s.device)[None, :] <= torch.arange(n, device=s.device)[:, None] + behind
        s = s.masked_fill(~see, -math.inf)
    return s


def _softmax(s):
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    return e / total, (top + torch.log(total))[..., 0]


def _plain_paged(st):
    case, out = st["case"], torch.zeros_like(st["q"])
    for s, (n, p, f) in enumerate(zip(st["new"], st["past"], st["first"])):
        pages = st["table"][s, :-(-(n + p) // case["page"])].long()
        k, v = (x[pages].transpose(0, 1).reshape(case["kv_heads"], -1, case["dim"])[:, :n + p].float()
                for x in (st["k_pages"], st["v_pages"]))
        q = st["q"][f:f + n].transpose(0, 1).float().contiguous()
        w, _ = _softmax(_scores(q, k, st["scale"], p))
        o = torch.matmul(w, v.repeat_interleave(q.shape[0] // v.shape[0], 0))
        out[f:f + n] = o.transpose(0, 1).to(out.dtype)
    return [out]


def _plain_prompt(st, train):
    case = st["case"]
    g, d, scale = case["heads"] // case["kv_heads"], case["dim"], st["scale"]
    out = torch.zeros_like(st["q"])
    lse = torch.zeros(st["rows"], case["heads"], dtype=torch.float32, device=out.device)
    grads = [torch.zeros_like(st[x]) for x in "qkv"] if train else []
    for n, f in zip(st["new"], st["first"]):
        q, k, v = (st[x][f:f + n].transpose(0, 1).float().contiguous() for x in "qkv")
        w, l = _softmax(_scores(q, k, scale, 0 if case["causal"] else None))
        vg = v.repeat_interleave(g, 0)
        o = torch.matmul(w, vg)
        out[f:f + n] = o.transpose(0, 1).to(out.dtype)
        lse[f:f + n] = l.transpose(0, 1)
        if train:
            do = st["dout"][f:f + n].transpose(0, 1).float().contiguous()
            dv = torch.matmul(w.transpose(1, 2).contiguous(), do)
            dw = torch.matmul(do, vg.transpose(1, 2).contiguous())
            ds = w * (dw - (do * o).sum(-1, keepdim=True)) * scale
            dq = torch.matmul(ds, k.repeat_interleave(g, 0))
            dk = torch.matmul(ds.transpose(1, 2).contiguous(), q)
            grads[0][f:f + n] = dq.transpose(0, 1).to(out.dtype)
            grads[1][f:f + n] = dk.reshape(-1, g, n, d).sum(1).transpose(0, 1).to(out.dtype)
            grads[2][f:f + n] = dv.reshape(-1, g, n, d).sum(1).transpose(0, 1).to(out.dtype)
    return [out] + grads if train else [out, lse]


# --------------------------------------------------------- the framework's calls
def _run_own(st):
    from futhark_amd.kernels import heads
    case, K, t = st["case"], st["K"], st["t"]
    h, hk, d, m, rows = case["heads"], case["kv_heads"], case["dim"], len(st["new"]), st["rows"]
    stream = torch.cuda.current_stream().cuda_stream

    def view(x):
        return heads(x.data_ptr(), x.stride(0), x.stride(1))

    seg = (st["offsets"].data_ptr(), st["lens"].data_ptr())
    fail = (st["failure"].data_ptr(), 1)
    if case["kind"] in ("append", "paged"):
        cache = (st["k_pages"].data_ptr(), st["v_pages"].data_ptr(), st["pages"], case["page"],
                 st["table"].data_ptr(), st["cols"])
    if case["kind"] == "append":
        K.kv_append(stream, t, view(st["q"]), view(st["out"]), view(st["k"]), view(st["v"]), rows, h, hk, d,
                    *seg, m, st["past_lens"].data_ptr(), st["freqs"].data_ptr(), case["rot"],
                    int(case["interleaved"]), *cache, *fail)
        return [st["out"], st["k_pages"], st["v_pages"]]
    if case["kind"] == "paged":
        K.attention_paged(stream, t, view(st["q"]), rows, h, hk, d, *seg, m, st["past_lens"].data_ptr(),
                          st["scale"], *cache, view(st["out"]), None, st["workspace"].data_ptr(),
                          st["workspace_bytes"], *fail)
        return [st["out"]]
    K.attention(stream, t, view(st["q"]), rows, view(st["k"]), view(st["v"]), rows, h, hk, d, *seg, *seg, m,
                st["scale"], int(case["causal"]), view(st["out"]), st["lse"].data_ptr(), *fail)
    if case["kind"] == "prompt":
        return [st["out"], st["lse"]]
    K.attention_grad(stream, t, view(st["q"]), rows, view(st["k"]), view(st["v"]), rows, h, hk, d, *seg, *seg, m,
                     st["scale"], int(case["causal"]), view(st["out"]), st["lse"].data_ptr(), view(st["dout"]),
                     view(st["dq"]), view(st["dk"]), view(st["dv"]), st["workspace"].data_ptr(),
                     st["workspace_bytes"], *fail)
    return [st["out"], st["dq"], st["dk"], st["dv"]]


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "append":
        return _plain_append(state)
    if kind == "paged":
        return _plain_paged(state)
    return _plain_prompt(state, kind == "train")


# ------------------------------------------------------- from the definition, in 64 bits
def _attend64(q, k, v, scale, behind):
    """One query head: q [n][dim] against k, v [keys][dim]; output and log of the sum."""
    s = (q @ k.T) * scale
    if behind is not None:
        i = torch.arange(s.shape[0], device=s.device).unsqueeze(1)
        j = torch.arange(s.shape[1], device=s.device).unsqueeze(0)
        s = torch.where(j > i + behind, torch.full_like(s, -math.inf), s)
    lse = torch.logsumexp(s, dim=1)
    return torch.exp(s - lse.unsqueeze(1)) @ v, lse


def exact(case, seed):
    st = _inputs(case, seed)
    g = case["heads"] // case["kv_heads"]
    if case["kind"] == "append":
        page, rot, half = case["page"], case["rot"], case["rot"] // 2
        q, k = st["q"].double(), st["k"].double()
        kp, vp = st["k_pages"].double(), st["v_pages"].double()
        if case["interleaved"]:
            first, second = torch.arange(0, rot, 2), torch.arange(1, rot, 2)
        else:
            first, second = torch.arange(half), torch.arange(half, rot)
        for s, (n, p, f) in enumerate(zip(st["new"], st["past"], st["first"])):
            where = torch.arange(p, p + n, device=q.device)
            turn = torch.polar(torch.ones(n, 1, half, dtype=torch.float64, device=q.device),
                               where.double().view(n, 1, 1) * st["freqs"].double())
            for x in (q, k):
                z = torch.complex(x[f:f + n][..., first], x[f:f + n][..., second]) * turn
                x[f:f + n, :, first], x[f:f + n, :, second] = z.real, z.imag
            at = st["table"][s].long()[torch.div(where, page, rounding_mode="floor")]
            kp[at, :, where % page] = k[f:f + n]
            vp[at, :, where % page] = st["v"][f:f + n].double()
        return [q, kp, vp]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    if case["kind"] == "paged":
        for s, (n, p, f) in enumerate(zip(st["new"], st["past"], st["first"])):
            pages = st["table"][s, :-(-(n + p) // case["page"])].long()
            for h in range(case["heads"]):
                k, v = (x[pages, h // g].reshape(-1, case["dim"])[:n + p].double()
                        for x in (st["k_pages"], st["v_pages"]))
                out[f:f + n, h], _ = _attend64(st["q"][f:f + n, h].double(), k, v, st["scale"], p)
        return [out]
    train = case["kind"] == "train"
    lse = torch.zeros(st["rows"], case["heads"], dtype=torch.float64, device=out.device)
    grads = [torch.zeros(st[x].shape, dtype=torch.float64, device=out.device) for x in "qkv"]
    behind = 0 if case["causal"] else None
    for n, f in zip(st["new"], st["first"]):
        for h in range(case["heads"]):
            q, k, v = (st[x][f:f + n, i].double().requires_grad_(train)
                       for x, i in (("q", h), ("k", h // g), ("v", h // g)))
            o, l = _attend64(q, k, v, st["scale"], behind)
            out[f:f + n, h], lse[f:f + n, h] = o.detach(), l.detach()
            if train:
                parts = torch.autograd.grad(o, (q, k, v), st["dout"][f:f + n, h].double())
                for whole, part, i in zip(grads, parts, (h, h // g, h // g)):
                    whole[f:f + n, i] += part
    return [out] + grads if train else [out, lse]
