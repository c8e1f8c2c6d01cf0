"""One step of speculative decoding, operator by operator: what is measured of it.

A drafter proposes a tree of tokens; the model evaluates all of them in one pass and keeps the path that its own sampled
tokens take. Around the projections (perf/cases.py) that step is four operators, each a call of the C ABI bound in
sardyne_amd.capi:

- "rope": rotary positions of tokens that do not stand one after another, their K/V rows written to slots;
- "attn": attention of the tree's nodes over the cache and over their own ancestors;
- "sample": a token per row of logits by temperature, top-k, top-p and min-p, from given uniform numbers;
- "commit": the walk along the sampled tokens and the accepted rows' copy into every layer's cache.

Sizes are those of the benchmark's 3B and 30B-A3B shapes (16 heads on 2, 32 on 4, head_dim 128, 36 and 48 layers,
vocabulary 151936), and generic ones.
"""
import ctypes
import math

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-6
KV = {"f32": (0, torch.float32, 4), "f16": (1, torch.float16, 2)}


# ------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one decoded token of the 3B shape: the smallest rotary call
        _rope("rope_1", 1, 16, 2, 128, 128, False, False, "f32", "none", 513),
        # a drafted tree of a 30B-A3B step: nodes of one depth share their position, rows go to the draft's own buffer
        _rope("rope_tree_61", 61, 32, 4, 128, 128, False, True, "f16", "yarn", 9000, tree=True),
        # a prompt chunk far into a long context, half of each head rotated, in the llama layout
        _rope("rope_prompt_2048", 2048, 32, 8, 128, 64, True, False, "f32", "llama3", 100_000),
        # a short draft in a chat: latency
        _attn("attn_5_700", 5, 700, 16, 2, 128, "f32"),
        # a full tree over a few pages of text
        _attn("attn_61_4099", 61, 4099, 32, 4, 128, "f32"),
        # a middling tree at the end of a long document, half-precision cache
        _attn("attn_24_33001_f16", 24, 33001, 16, 2, 128, "f16"),
        # a full tree over a long document
        _attn("attn_64_40000", 64, 40000, 32, 4, 128, "f32"),
        # the token of a chat's decode step
        _sample("sample_1", 1, 151936, "chat", "float"),
        # every node of a drafted tree, requests of all kinds
        _sample("sample_61", 61, 151936, "mixed", "float"),
        # many rows of a smaller vocabulary under a grammar that leaves few tokens
        _sample("sample_250_grammar", 250, 32000, "mixed", "masked"),
        # a short draft's rows into the 3B shape's caches
        _commit("commit_8", 8, 36, 2, 128, "f32", 1024),
        # a full tree's into the 30B-A3B shape's
        _commit("commit_61", 61, 48, 4, 128, "f16", 2048),
    ]


def _rope(name, n_tok, n_head, n_kv_head, hd, n_rot, interleaved, qk_norm, kv, scaling, past, tree=False):
    return {"name": name, "kind": "rope", "n_tok": n_tok, "n_head": n_head, "n_kv_head": n_kv_head, "head_dim": hd,
            "n_rot": n_rot, "interleaved": interleaved, "qk_norm": qk_norm, "kv": kv, "scaling": scaling, "past": past,
            "tree": tree}


def _attn(name, n_tok, past, n_head, n_kv_head, hd, kv):
    return {"name": name, "kind": "attn", "n_tok": n_tok, "past": past, "n_head": n_head, "n_kv_head": n_kv_head,
            "head_dim": hd, "kv": kv}


def _sample(name, n_rows, n_vocab, params, logits):
    return {"name": name, "kind": "sample", "n_rows": n_rows, "n_vocab": n_vocab, "params": params, "logits": logits}


def _commit(name, n_tok, n_layer, n_kv_head, hd, kv, max_seq):
    return {"name": name, "kind": "commit", "n_tok": n_tok, "n_layer": n_layer, "n_kv_head": n_kv_head, "head_dim": hd,
            "kv": kv, "max_seq": max_seq}


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "attn", "attn", "attn", "attn", "sample", "sample", "sample", "commit"])
    n_kv_head = rng.choice([1, 2, 4, 8])
    n_head = n_kv_head * rng.choice([1, 2, 4, 7, 8] if n_kv_head < 8 else [1, 2, 4])
    hd, kv = rng.choice([64, 128, 128, 256]), rng.choice(["f32", "f16"])
    if kind == "rope":
        tree = rng.random() < 0.4
        return {"kind": kind, "n_tok": _log_int(rng, 1, 255 if tree else 1024), "n_head": min(n_head, 32),
                "n_kv_head": n_kv_head, "head_dim": hd, "n_rot": rng.choice([hd, hd, hd // 2, hd // 4, hd - 6]),
                "interleaved": rng.random() < 0.5, "qk_norm": rng.random() < 0.5, "kv": kv,
                "scaling": rng.choice(["none", "linear", "yarn", "llama3"]), "past": _log_int(rng, 1, 1_000_000),
                "tree": tree}
    if kind == "attn":
        n_tok = _log_int(rng, 1, 255)
        most = min(64 * 40000 * 32 * 128 // (n_tok * n_head * hd), 40000 * 4 * 128 // (n_kv_head * hd), 131072)
        return {"kind": kind, "n_tok": n_tok, "past": _log_int(rng, 1, most), "n_head": n_head, "n_kv_head": n_kv_head,
                "head_dim": hd, "kv": kv}
    if kind == "sample":
        n_vocab = _log_int(rng, 257, 151936)
        return {"kind": kind, "n_rows": _log_int(rng, 1, min(1024, 61 * 151936 // n_vocab)), "n_vocab": n_vocab,
                "params": rng.choice(["chat", "mixed", "plain"]), "logits": rng.choice(["float", "masked", "coarse"])}
    n_layer = rng.choice([1, 12, 28, 36, 48])
    return {"kind": kind, "n_tok": _log_int(rng, 1, 255), "n_layer": n_layer, "n_kv_head": n_kv_head,
            "head_dim": min(hd, 128), "kv": kv, "max_seq": _log_int(rng, 300, 300 + 60000 // (n_layer * n_kv_head))}


# ------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _tree(n_tok, rng):
    """Parents of a drafted tree: each node under one of the eight before it; the last few places of a tree of more than
    eight are unused (-2), as where a step of fixed size has fewer drafts."""
    parent = [-1] + [int(rng.integers(max(0, t - 8), t)) for t in range(1, n_tok)]
    if n_tok > 8:
        for t in range(n_tok - int(rng.integers(0, 4)), n_tok):
            parent[t] = -2
    return parent


def _depths(parent):
    depth = []
    for p in parent:
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return depth


def _frequencies(n_rot, scaling, theta=1e6, factor=8.0, orig=8192):
    """freq[i] of the rotation's pairs and the factor on cos and sin, by the published formulas."""
    i = np.arange(n_rot // 2)
    f = 1.0 / theta ** (2.0 * i / n_rot)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        turn = [n_rot * math.log(orig / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (32.0, 1.0)]
        low, high = max(math.floor(turn[0]), 0), min(math.ceil(turn[1]), n_rot - 1)
        ramp = np.clip((i - low) / max(high - low, 1e-3), 0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if scaling == "llama3":
        turns = orig * f / (2 * math.pi)
        smooth = np.clip((turns - 1.0) / (4.0 - 1.0), 0, 1)
        return f * ((1 - smooth) / factor + smooth), 1.0
    return f, 1.0


def _prepare_rope(case, seed):
    g, rng = _gen(seed), np.random.default_rng(seed)
    n, nh, nkv, hd = case["n_tok"], case["n_head"], case["n_kv_head"], case["head_dim"]
    qkv = _randn(g, n, (nh + 2 * nkv) * hd)  # rows of one stacked projection
    if case["tree"]:
        parent = _tree(n, rng)
        pos = [case["past"] + d for d in _depths(parent)]
        slot = [t if p > -2 else -1 for t, p in enumerate(parent)]
        n_slot = n
    else:
        pos = list(range(case["past"], case["past"] + n))
        slot = list(range(3, 3 + n))
        n_slot = n + 5
    freq, mscale = _frequencies(case["n_rot"], case["scaling"])
    _, dtype, _ = KV[case["kv"]]
    # one row more than there are slots, which no token names
    rows = [_randn(g, nkv, n_slot + 1, hd).to(dtype) for _ in range(2)]
    return {"case": case, "qkv": qkv, "pos": _i32(pos), "slot": _i32(slot), "n_slot": n_slot, "k_rows": rows[0],
            "v_rows": rows[1], "freq": torch.tensor(freq, dtype=torch.float64, device=DEV), "mscale": mscale,
            "q_norm": 1 + 0.1 * _randn(g, hd), "k_norm": 1 + 0.1 * _randn(g, hd),
            "q_out": torch.zeros(n, nh * hd, device=DEV)}


def _prepare_attn(case, seed):
    g, rng = _gen(seed), np.random.default_rng(seed)
    n, nh, nkv, hd, past = (case[k] for k in ("n_tok", "n_head", "n_kv_head", "head_dim", "past"))
    max_seq = past + 64
    _, dtype, _ = KV[case["kv"]]
    # keys with a few large dims and a few positions that most queries look at, as caches have them
    dims = 1 + 3 * (torch.rand(nkv, 1, hd, generator=g, device=DEV) < 0.03)
    sink = 1 + 0.5 * (torch.rand(nkv, max_seq, 1, generator=g, device=DEV) < 0.001)
    cache = [(_randn(g, nkv, max_seq, hd) * dims * sink).to(dtype), _randn(g, nkv, max_seq, hd).to(dtype)]
    draft = [(_randn(g, nkv, n, hd) * dims).to(dtype), _randn(g, nkv, n, hd).to(dtype)]
    return {"case": case, "q": 1.2 * _randn(g, n, nh * hd), "k_cache": cache[0], "v_cache": cache[1], "k_draft": draft[0],
            "v_draft": draft[1], "parent": _i32(_tree(n, rng)), "n_past": _i32([past]), "max_past": max_seq,
            "out": torch.zeros(n, nh * hd, device=DEV)}


def _prepare_sample(case, seed):
    g, rng = _gen(seed), np.random.default_rng(seed)
    n, v = case["n_rows"], case["n_vocab"]
    x = 2.0 * _randn(g, n, v)
    tail = torch.rand(n, v, generator=g, device=DEV).clamp_min(1e-7)
    x -= 1.3 * torch.log(tail)  # a few tokens stand out, as where a model knows what comes
    if case["logits"] == "masked":  # a grammar leaves a tenth of the vocabulary
        x[torch.rand(n, v, generator=g, device=DEV) < 0.9] = -math.inf
    if case["logits"] == "coarse":  # a half-precision head's ties
        x = x.to(torch.bfloat16).float()
    if case["params"] == "chat":
        temp, top_k, top_p, min_p = [0.7] * n, [20] * n, [0.8] * n, [0.0] * n
    elif case["params"] == "plain":
        temp, top_k, top_p, min_p = [1.0] * n, [0] * n, [1.0] * n, [0.0] * n
    else:
        temp = rng.choice([0.0, 0.6, 0.8, 1.0, 1.3], n)
        top_k, top_p = rng.choice([0, 20, 40, 400], n), rng.choice([0.8, 0.95, 1.0], n)
        min_p = rng.choice([0.0, 0.0, 0.05], n)
    f32 = lambda a: torch.tensor(np.asarray(a, np.float32), device=DEV)  # noqa: E731
    return {"case": case, "logits": x, "temp": f32(temp), "top_k": _i32([int(k) for k in top_k]), "top_p": f32(top_p),
            "min_p": f32(min_p), "u": torch.rand(n, generator=g, device=DEV),
            "token": torch.zeros(n, dtype=torch.int32, device=DEV), "prob": torch.zeros(n, device=DEV)}


def _prepare_commit(case, seed):
    g, rng = _gen(seed), np.random.default_rng(seed)
    n, nl, nkv, hd, max_seq = (case[k] for k in ("n_tok", "n_layer", "n_kv_head", "head_dim", "max_seq"))
    _, dtype, _ = KV[case["kv"]]
    parent = _tree(n, rng)
    token = rng.choice(151936, n, replace=False)
    children = {}
    for t, p in enumerate(parent):
        children.setdefault(p, []).append(t)
    # the model agrees with one of a node's drafts about four times in five
    sampled = [int(token[rng.choice(children[t])]) if t in children and rng.random() < 0.8 else
               int(rng.integers(0, 151936)) for t in range(n)]
    make = lambda *s: _randn(g, *s).to(dtype)  # noqa: E731
    return {"case": case, "token": _i32([int(t) for t in token]), "parent": _i32(parent), "sampled": _i32(sampled),
            "n_past": _i32([int(rng.integers(1, max_seq - n + 1))]), "k_draft": make(nl, nkv, n, hd),
            "v_draft": make(nl, nkv, n, hd), "k_cache": make(nl, nkv, max_seq, hd), "v_cache": make(nl, nkv, max_seq, hd),
            "path": torch.zeros(n, dtype=torch.int32, device=DEV), "n_acc": torch.zeros(1, dtype=torch.int32, device=DEV),
            "step": torch.zeros(2, dtype=torch.int32, device=DEV)}


def prepare(case, seed):
    return {"rope": _prepare_rope, "attn": _prepare_attn, "sample": _prepare_sample,
            "commit": _prepare_commit}[case["kind"]](case, seed)


# -------------------------------------------------------------------------------------- plain forms

def _split_heads(s):
    c = s["case"]
    nh, nkv, hd = c["n_head"], c["n_kv_head"], c["head_dim"]
    q, k, v = s["qkv"].split([nh * hd, nkv * hd, nkv * hd], 1)
    return q.view(-1, nh, hd), k.view(-1, nkv, hd), v.view(-1, nkv, hd)


def _plain_rope(s):
    c = s["case"]
    rot, half = c["n_rot"], c["n_rot"] // 2
    q, k, v = _split_heads(s)
    if c["qk_norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"]
    angle = s["pos"].double()[:, None, None] * s["freq"]
    cos, sin = (s["mscale"] * angle.cos()).float(), (s["mscale"] * angle.sin()).float()

    def rotate(x):
        x = x.clone()
        if c["interleaved"]:
            a, b = x[..., 0:rot:2].clone(), x[..., 1:rot:2].clone()
            x[..., 0:rot:2], x[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
        else:
            a, b = x[..., :half].clone(), x[..., half:rot].clone()
            x[..., :half], x[..., half:rot] = a * cos - b * sin, a * sin + b * cos
        return x

    at = s["slot"].long()  # -1, no slot, is the row behind the last one
    s["k_rows"][:, at] = rotate(k).transpose(0, 1).to(s["k_rows"].dtype)
    s["v_rows"][:, at] = v.transpose(0, 1).to(s["v_rows"].dtype)
    s["q_out"].copy_(rotate(q).flatten(1))
    return _rope_out(s)


def _rope_out(s):
    return {"q": s["q_out"], "k": s["k_rows"][:, :s["n_slot"]], "v": s["v_rows"][:, :s["n_slot"]]}


def _ancestors(parent):
    """[n][n]: whether node j is node t or above it. (I + P)^256 counts the ways up."""
    n = parent.numel()
    up = (parent[:, None] == torch.arange(n, device=DEV)).double()
    return torch.linalg.matrix_power(torch.eye(n, dtype=torch.float64, device=DEV) + up, 256) > 0


def _plain_attn(s):
    c = s["case"]
    n, nh, nkv, hd = c["n_tok"], c["n_head"], c["n_kv_head"], c["head_dim"]
    past, rep = c["past"], nh // nkv
    k = torch.cat([s["k_cache"][:, :past], s["k_draft"]], 1).float()
    v = torch.cat([s["v_cache"][:, :past], s["v_draft"]], 1).float()
    q = s["q"].view(n, nkv, rep, hd).permute(1, 0, 2, 3).reshape(nkv, n * rep, hd) / math.sqrt(hd)
    score = torch.matmul(q, k.transpose(1, 2).contiguous()).view(nkv, n, rep, past + n)
    sees = torch.cat([torch.ones(n, past, dtype=torch.bool, device=DEV), _ancestors(s["parent"])], 1)
    score.masked_fill_(~sees[None, :, None, :], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(nkv, n * rep, past + n)
    o = torch.matmul(p, v).view(nkv, n, rep, hd).permute(1, 0, 2, 3).reshape(n, nh * hd)
    s["out"].copy_(torch.where((s["parent"] > -2)[:, None], o, s["out"]))
    return s["out"]


def _plain_sample(s):
    x = s["logits"].double()
    x = torch.where(x.isnan(), -math.inf, x)
    n, v = x.shape
    best, first = x.max(1, keepdim=True)
    first = torch.where(x == best, torch.arange(v, device=DEV), v).amin(1, keepdim=True)
    greedy = ~(s["temp"] > 0)[:, None]
    t = torch.where(greedy[:, 0], 1.0, s["temp"])[:, None].double()
    w = torch.where(x == best, 1.0, torch.where(x == -math.inf, 0.0, torch.exp((x - best) / t)))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    k = torch.where(s["top_k"] > 0, s["top_k"].long(), v)[:, None]
    rank = torch.arange(v, device=DEV)
    wk = torch.where(rank < k, ws, 0.0)
    before = torch.cumsum(wk, 1) - wk
    keep = (rank < k) & (before < s["top_p"][:, None].double() * wk.sum(1, keepdim=True)) & \
        (ws >= s["min_p"][:, None].double()) | (rank == 0)
    kept = torch.zeros(n, v, dtype=torch.float64, device=DEV).scatter_(1, order, torch.where(keep, ws, 0.0))
    kept = torch.where(greedy, (torch.arange(v, device=DEV) == first).double(), kept)
    run_sum = torch.cumsum(kept, 1)
    total = run_sum[:, -1:]
    token = (run_sum <= s["u"][:, None].double() * total).sum(1, keepdim=True).clamp_max(v - 1)
    s["token"].copy_(token[:, 0])
    s["prob"].copy_((kept.gather(1, token) / total)[:, 0])
    return {"token": s["token"], "prob": s["prob"]}


def _plain_commit(s):
    token, parent, sampled = s["token"], s["parent"].long(), s["sampled"]
    n = token.numel()
    at = torch.arange(n, device=DEV)
    up = parent.clamp_min(0)
    fits = (parent >= 0) & (token == sampled[up])
    twin = (fits[:, None] & fits[None, :] & (parent[:, None] == parent[None, :]) & (at[None, :] < at[:, None])).any(1)
    fits = (fits & ~twin) | (at == 0)
    accepted = ~(_ancestors(s["parent"]) & ~fits[None, :]).any(1)
    count = accepted.sum()
    path = torch.where(accepted, at, n).sort().values
    last = path[count - 1]
    path = torch.where(at < count, path, -1)
    s["path"].copy_(path)
    s["n_acc"].copy_(count[None])
    s["step"].copy_(torch.stack([sampled[last], s["n_past"][0] + count]))
    to = s["n_past"].long() + at
    took = (at < count)[:, None]
    node = path.clamp_min(0)
    s["k_cache"][:, :, to] = torch.where(took, s["k_draft"][:, :, node], s["k_cache"][:, :, to])
    s["v_cache"][:, :, to] = torch.where(took, s["v_draft"][:, :, node], s["v_cache"][:, :, to])
    return _commit_out(s)


def _commit_out(s):
    return {k: s[k] for k in ("path", "n_acc", "step", "k_cache", "v_cache")}


# ---------------------------------------------------------------------------------- the framework's

def _own_rope(s):
    from sardyne_amd import capi
    c, lib = s["case"], capi.lib()
    if "args" not in s:
        capi.check(lib.sdy_init())
        q, k, v = (x.data_ptr() for x in _split_heads(s))
        stride, norm = s["qkv"].shape[1], c["qk_norm"]
        s["args"] = capi.SdyRopeAtArgs(
            q=q, k=k, v=v, q_stride=stride, k_stride=stride, v_stride=stride, q_out=s["q_out"].data_ptr(),
            q_out_stride=s["q_out"].shape[1], k_rows=s["k_rows"].data_ptr(), v_rows=s["v_rows"].data_ptr(),
            head_stride=s["k_rows"].stride(0), kv_type=KV[c["kv"]][0], n_slot=s["n_slot"], pos=s["pos"].data_ptr(),
            slot=s["slot"].data_ptr(), freq=s["freq"].data_ptr(), mscale=s["mscale"], n_rot=c["n_rot"],
            interleaved=int(c["interleaved"]), q_norm=s["q_norm"].data_ptr() if norm else None,
            k_norm=s["k_norm"].data_ptr() if norm else None, eps=EPS, n_tok=c["n_tok"], n_head=c["n_head"],
            n_kv_head=c["n_kv_head"], hd=c["head_dim"])
    capi.check(lib.sdy_qk_rope_at(ctypes.byref(s["args"]), None))
    return _rope_out(s)


def _own_attn(s):
    from sardyne_amd import capi
    c, lib = s["case"], capi.lib()
    if "args" not in s:
        capi.check(lib.sdy_init())
        floats = lib.sdy_attn_tree_floats(c["n_tok"], c["n_head"], c["n_kv_head"], c["head_dim"], s["max_past"])
        s["part"] = torch.empty(floats, device=DEV)
        s["args"] = capi.SdyAttnTreeArgs(
            q=s["q"].data_ptr(), q_stride=s["q"].shape[1], k_cache=s["k_cache"].data_ptr(),
            v_cache=s["v_cache"].data_ptr(), head_stride=s["k_cache"].stride(0), k_draft=s["k_draft"].data_ptr(),
            v_draft=s["v_draft"].data_ptr(), draft_stride=s["k_draft"].stride(0), kv_type=KV[c["kv"]][0],
            parent=s["parent"].data_ptr(), n_past=s["n_past"].data_ptr(), max_past=s["max_past"], n_tok=c["n_tok"],
            n_head=c["n_head"], n_kv_head=c["n_kv_head"], hd=c["head_dim"], out=s["out"].data_ptr(),
            out_stride=s["out"].shape[1], part=s["part"].data_ptr())
    capi.check(lib.sdy_attn_tree(ctypes.byref(s["args"]), None))
    return s["out"]


def _own_sample(s):
    from sardyne_amd import capi
    c, lib = s["case"], capi.lib()
    if "args" not in s:
        capi.check(lib.sdy_init())
        s["ws"] = torch.empty(lib.sdy_sample_ws_bytes(c["n_rows"], c["n_vocab"]), dtype=torch.uint8, device=DEV)
        s["args"] = capi.SdySampleArgs(
            logits=s["logits"].data_ptr(), stride=s["logits"].shape[1], n_rows=c["n_rows"], n_vocab=c["n_vocab"],
            temp=s["temp"].data_ptr(), top_k=s["top_k"].data_ptr(), top_p=s["top_p"].data_ptr(),
            min_p=s["min_p"].data_ptr(), u=s["u"].data_ptr(), token=s["token"].data_ptr(), prob=s["prob"].data_ptr(),
            ws=s["ws"].data_ptr())
    capi.check(lib.sdy_sample(ctypes.byref(s["args"]), None))
    return {"token": s["token"], "prob": s["prob"]}


def _own_commit(s):
    from sardyne_amd import capi
    c, lib = s["case"], capi.lib()
    if "args" not in s:
        capi.check(lib.sdy_init())
        s["args"] = capi.SdyTreeCommitArgs(
            token=s["token"].data_ptr(), parent=s["parent"].data_ptr(), sampled=s["sampled"].data_ptr(),
            n_tok=c["n_tok"], n_past=s["n_past"].data_ptr(), k_draft=s["k_draft"].data_ptr(),
            v_draft=s["v_draft"].data_ptr(), draft_stride=s["k_draft"].stride(1),
            draft_layer_stride=s["k_draft"].stride(0), k_cache=s["k_cache"].data_ptr(), v_cache=s["v_cache"].data_ptr(),
            head_stride=s["k_cache"].stride(1), layer_stride=s["k_cache"].stride(0), kv_type=KV[c["kv"]][0],
            max_seq=c["max_seq"], n_layer=c["n_layer"], n_kv_head=c["n_kv_head"], hd=c["head_dim"],
            path=s["path"].data_ptr(), n_acc=s["n_acc"].data_ptr(), step=s["step"].data_ptr())
    capi.check(lib.sdy_tree_commit(ctypes.byref(s["args"]), None))
    return _commit_out(s)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rope": _own_rope, "attn": _own_attn, "sample": _own_sample, "commit": _own_commit}[kind](state)
    return {"rope": _plain_rope, "attn": _plain_attn, "sample": _plain_sample, "commit": _plain_commit}[kind](state)


# -------------------------------------------------------------------------------------------- work

def work(case):
    n, kind = case.get("n_tok"), case["kind"]
    if kind == "sample":
        size = case["n_rows"] * case["n_vocab"]
        return {"bytes": 4 * size + 28 * case["n_rows"], "flops": 4 * size}  # difference, exp, sum, comparison
    nkv, hd, elt = case["n_kv_head"], case["head_dim"], KV[case["kv"]][2]
    if kind == "rope":
        nh = case["n_head"]
        values = n * (nh + nkv) * hd
        return {"bytes": 8 * n * nh * hd + 2 * n * nkv * hd * (4 + elt) + 8 * n, "flops": 3 * values}
    if kind == "attn":
        nh, past = case["n_head"], case["past"]
        pairs = n * past + sum(_about_depth(t) for t in range(n))
        return {"bytes": 2 * nkv * (past + n) * hd * elt + 8 * n * nh * hd + 4 * n, "flops": 4 * nh * hd * pairs}
    # the accepted path's rows, four nodes of a tree or so, read and written
    rows = min(n, 4)
    return {"bytes": 4 * case["n_layer"] * nkv * rows * hd * elt + 16 * n, "flops": n}


def _about_depth(t):
    return 1 + (t + 3) // 5  # parents are about 4.5 places back


# ---------------------------------------------------------------------------------- from definitions

def _exact_rope(case, seed):
    s = _prepare_rope(case, seed)
    rot, hd, n = case["n_rot"], case["head_dim"], case["n_tok"]
    nh, nkv = case["n_head"], case["n_kv_head"]
    x = s["qkv"].double().view(n, nh + 2 * nkv, hd)
    q, k, v = x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]
    if case["qk_norm"]:
        q = q / ((q * q).sum(-1, keepdim=True) / hd + EPS).sqrt() * s["q_norm"].double()
        k = k / ((k * k).sum(-1, keepdim=True) / hd + EPS).sqrt() * s["k_norm"].double()
    # a rotation by a complex number of length mscale
    turn = torch.polar(torch.full_like(s["freq"], s["mscale"]).expand(n, -1).contiguous(),
                       s["pos"].double()[:, None] * s["freq"][None, :])[:, None, :]
    first = torch.arange(rot // 2, device=DEV)
    re, im = (2 * first, 2 * first + 1) if case["interleaved"] else (first, first + rot // 2)

    def turned(y):
        z = torch.complex(y[..., re].contiguous(), y[..., im].contiguous()) * turn
        y = y.clone()
        y[..., re], y[..., im] = z.real, z.imag
        return y

    out = {"q": turned(q).reshape(n, nh * hd), "k": s["k_rows"][:, :-1].double(), "v": s["v_rows"][:, :-1].double()}
    tk = turned(k)
    for t, at in enumerate(s["slot"].tolist()):
        if at >= 0:
            out["k"][:, at], out["v"][:, at] = tk[t], v[t]
    return out


def _exact_attn(case, seed):
    s = _prepare_attn(case, seed)
    n, nh, nkv, hd, past = (case[k] for k in ("n_tok", "n_head", "n_kv_head", "head_dim", "past"))
    parent = s["parent"].tolist()
    sees = torch.zeros(n, n, dtype=torch.bool, device=DEV)
    for t in range(n):
        u = t
        while u >= 0:
            sees[t, u] = True
            u = parent[u]
    out = torch.zeros(n, nh, hd, dtype=torch.float64, device=DEV)
    used = torch.tensor([p > -2 for p in parent], device=DEV)
    for h in range(nh):
        g = h // (nh // nkv)
        q = s["q"].view(n, nh, hd)[:, h].double()
        a = q @ s["k_cache"][g, :past].double().T.contiguous() * hd ** -0.5
        b = (q @ s["k_draft"][g].double().T.contiguous() * hd ** -0.5).masked_fill(~sees, -math.inf)
        z = torch.logsumexp(torch.cat([a, b], 1), 1, keepdim=True)
        o = torch.exp(a - z) @ s["v_cache"][g, :past].double() + torch.exp(b - z) @ s["v_draft"][g].double()
        out[:, h] = torch.where(used[:, None], o, 0.0)
    return out.view(n, nh * hd)


def _exact_sample(case, seed):
    s = _prepare_sample(case, seed)
    x = s["logits"].cpu().numpy().astype(np.float64)
    temp, top_k, top_p, min_p, u = (s[k].cpu().numpy().astype(np.float64) for k in ("temp", "top_k", "top_p", "min_p", "u"))
    tokens, probs = [], []
    for r in range(case["n_rows"]):
        if temp[r] <= 0:
            tokens.append(int(np.argmax(x[r])))
            probs.append(1.0)
            continue
        order = np.argsort(-x[r], kind="stable")
        if top_k[r] > 0:
            order = order[:int(top_k[r])]
        w = np.exp((x[r][order] - x[r][order[0]]) / temp[r])
        n = len(order)
        if top_p[r] < 1:
            n = 1 + int(np.searchsorted(np.cumsum(w), top_p[r] * w.sum()))
        n = max(1, min(n, int(np.searchsorted(-w, -min_p[r], side="right"))))
        kept = np.sort(order[:n])
        w = np.exp((x[r][kept] - x[r][order[0]]) / temp[r])
        at = min(int(np.searchsorted(np.cumsum(w), u[r] * w.sum(), side="right")), n - 1)
        tokens.append(int(kept[at]))
        probs.append(float(w[at] / w.sum()))
    return {"token": torch.tensor(tokens, dtype=torch.int32), "prob": torch.tensor(probs, dtype=torch.float64)}


def _exact_commit(case, seed):
    s = _prepare_commit(case, seed)
    token, parent, sampled, past = (s[k].tolist() for k in ("token", "parent", "sampled", "n_past"))
    path = [0]
    while True:
        nxt = [t for t, p in enumerate(parent) if p == path[-1] and token[t] == sampled[path[-1]]]
        if not nxt:
            break
        path.append(nxt[0])
    out = {"path": _i32(path + [-1] * (len(token) - len(path))), "n_acc": _i32([len(path)]),
           "step": _i32([sampled[path[-1]], past[0] + len(path)])}
    for name in ("k", "v"):
        out[name + "_cache"] = s[name + "_cache"].double()
        for i, t in enumerate(path):
            out[name + "_cache"][:, :, past[0] + i] = s[name + "_draft"][:, :, t].double()
    return out


def exact(case, seed):
    return {"rope": _exact_rope, "attn": _exact_attn, "sample": _exact_sample, "commit": _exact_commit}[case["kind"]](case, seed)
