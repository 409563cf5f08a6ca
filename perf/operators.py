"""Measured cases of the operators over a paged KV cache: attention of packed
chunks of new tokens, the attention weight each cached key has received, and
eviction of the keys that received least.

Each operator is here in a plain form (elementary torch operations in 32 bits)
and as the calls a user of the library makes.  A cache is f16 or bf16 pages
[page][kv_head][64][head_dim] behind a block table; head shapes are those of
the library's own configurations (0.5B: 14/2 heads of 64; 1.5B: 12/2 of 128;
7B: 28/4 of 128) and a few generic ones."""
import math
import random
import sys
from pathlib import Path

import torch

own = False

PAGE = 64
DEV = "cuda:0"
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _vvq2():
    pkg = str(Path(__file__).resolve().parent.parent / "vibevoice.cpp_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import vvq2
    return vvq2


# ------------------------------------------------------------------ cases
def _attn(name, n_seqs, q, past, heads, dtype="f16", lens=1):
    """q, past: (lowest, highest) new tokens and keys already cached of a sequence."""
    nq, nkv, hd = heads
    c = {"op": "attention", "n_seqs": n_seqs, "q_lo": q[0], "q_hi": q[1], "past_lo": past[0], "past_hi": past[1],
         "nq": nq, "nkv": nkv, "hd": hd, "dtype": dtype, "lens": lens}
    return dict(c, name=name) if name else c


def _weights(name, n_seqs, q, past, heads, dtype="f16", lens=1, fresh=False):
    """fresh: the chunk's weights alone; else they are added to the older keys'."""
    return dict(_attn(name, n_seqs, q, past, heads, dtype, lens), op="weights", fresh=fresh)


def _evict(name, layers, n_seqs, length, keep, first, recent, nkv, hd, dtype="f16", lens=1):
    c = {"op": "evict", "layers": layers, "n_seqs": n_seqs, "len_lo": length[0], "len_hi": length[1], "keep": keep,
         "first": first, "recent": recent, "nkv": nkv, "hd": hd, "dtype": dtype, "lens": lens}
    return dict(c, name=name) if name else c


S, M, L = (14, 2, 64), (12, 2, 128), (28, 4, 128)


def listed():
    return [
        # one frame of a guided stream: a conditional and an unconditional row, 1024 keys each
        _attn("attend-decode-pair", 2, (1, 1), (1023, 1023), S),
        # one decode step of 64 guided streams of different age
        _attn("attend-decode-128-ragged", 128, (1, 1), (63, 2047), S),
        # one decode step far into a long transcription
        _attn("attend-decode-27k", 1, (1, 1), (27000, 27000), L),
        # a few drafted tokens per stream checked at once, bf16 pages
        _attn("attend-draft-ragged", 12, (2, 9), (17, 5003), M, "bf16"),
        # prompts of different lengths prefilled in one packed call
        _attn("attend-prompts-packed", 24, (1, 2047), (0, 0), S),
        # a whole long prompt
        _attn("attend-prompt-16k", 1, (16384, 16384), (0, 0), L),
        # weights updated after a decode step of a batch of streams
        _weights("weigh-decode-ragged", 64, (1, 1), (63, 2047), S),
        # the last questions of a long prompt decide what the cache keeps
        _weights("weigh-window-16k", 1, (32, 32), (16352, 16352), L, fresh=True),
        # weights of packed prompts, each query counted, bf16 pages
        _weights("weigh-prompts-packed", 6, (131, 4001), (0, 500), M, "bf16"),
        # one layer of a guided pair cut back to half its window
        _evict("evict-pair", 1, 2, (1100, 1101), 512, 108, 128, 2, 64),
        # all layers of a ragged batch, some sequences below the budget
        _evict("evict-batch-24-layers", 24, 16, (190, 2048), 700, 64, 65, 2, 64, "bf16"),
        # all layers of one long transcription
        _evict("evict-27k-28-layers", 28, 1, (27000, 27000), 8192, 128, 1024, 4, 128),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _draw(rng):
    heads = rng.choice([S, M, L, (8, 8, 64), (8, 1, 128), (20, 4, 64)])
    dtype = rng.choice(["f16", "f16", "bf16"])
    lens = rng.randrange(1, 1 << 20)
    op = rng.choice(["decode", "draft", "prompts", "chunk", "weights", "weights-decode", "evict"])
    if op == "evict":
        n = _log(rng, 1, 32)
        hi = _log(rng, 65, 27000)
        lo = rng.randint(max(1, hi // 8), hi)
        keep = _log(rng, 16, max(17, hi))
        first = rng.randint(0, keep // 4)
        recent = rng.randint(0, keep // 3)
        return _evict(None, rng.randint(1, 28), n, (lo, hi), keep, first, recent, heads[1], heads[2], dtype, lens)
    if op in ("decode", "weights-decode"):
        hi = _log(rng, 1, 32000)
        n, q, past = _log(rng, 1, 160), (1, 1), (rng.randint(0, hi), hi)
    elif op == "draft":
        hi = _log(rng, 1, 20000)
        q_hi = rng.randint(2, 24)
        n, q, past = _log(rng, 1, 64), (rng.randint(1, q_hi), q_hi), (rng.randint(0, hi), hi)
    elif op == "prompts":
        hi = _log(rng, 8, 12000)
        n, q, past = _log(rng, 1, 48), (rng.randint(1, hi), hi), (0, 0)
    else:
        hi, p = _log(rng, 16, 6000), _log(rng, 1, 20000)
        n, q, past = _log(rng, 1, 8), (rng.randint(1, hi), hi), (rng.randint(0, p), p)
    if op.startswith("weights"):
        return _weights(None, n, q, past, heads, dtype, lens, rng.random() < 0.3)
    return _attn(None, n, q, past, heads, dtype, lens)


def draw(rng):
    """One more case, no dearer than the dearest listed one of its operator."""
    top = {}
    for c in listed():
        w, t = work(c), top.setdefault(c["op"], {"bytes": 0, "flops": 0, "keys": 0})
        for k in w:
            t[k] = max(t[k], w[k])
        t["keys"] = max(t["keys"], _padded_keys(c))
    while True:
        c = _draw(rng)
        w, t = work(c), top[c["op"]]
        if w["bytes"] <= t["bytes"] and w["flops"] <= t["flops"] and _padded_keys(c) <= t["keys"]:
            return c


def _lengths(case):
    """[(new tokens, cached keys with them)] of an attention case, [length] of an eviction."""
    r = random.Random(case["lens"])
    if case["op"] == "evict":
        return [r.randint(case["len_lo"], case["len_hi"]) for _ in range(case["n_seqs"])]
    out = []
    for _ in range(case["n_seqs"]):
        n = r.randint(case["q_lo"], case["q_hi"])
        out.append((n, n + r.randint(case["past_lo"], case["past_hi"])))
    return out


def _padded_keys(case):
    """Bound on what a batch padded to its longest sequence holds."""
    if case["op"] == "evict":
        return case["layers"] * case["n_seqs"] * case["len_hi"] * case["nkv"] * case["hd"]
    return case["n_seqs"] * (case["q_hi"] + case["past_hi"]) * case["nkv"] * case["hd"]


def _pairs(ls):
    """Visible (token, key) pairs."""
    return sum(n * (kv - n) + n * (n + 1) // 2 for n, kv in ls)


def work(case):
    nkv, hd = case["nkv"], case["hd"]
    ls = _lengths(case)
    if case["op"] == "evict":
        keep = sum(min(l, case["keep"]) for l in ls)
        by = case["layers"] * nkv * (4 * sum(ls) + keep * (2 * 2 * hd * 2 + 4 + 4)) + 8 * len(ls)
        return {"bytes": by, "flops": 0}
    nq, total, keys = case["nq"], sum(n for n, _ in ls), sum(kv for _, kv in ls)
    if case["op"] == "attention":
        return {"bytes": 2 * 2 * keys * nkv * hd + 2 * 2 * total * nq * hd + 4 * total * nq,
                "flops": 4 * nq * hd * _pairs(ls)}
    old = 0 if case["fresh"] else sum(kv - n for n, kv in ls)
    return {"bytes": 2 * keys * nkv * hd + 2 * total * nq * hd + 4 * total * nq + 4 * nkv * (keys + old),
            "flops": 2 * nq * hd * _pairs(ls)}


# ----------------------------------------------------------------- inputs
def _table(lens, gen, first_page=0):
    """Block table of sequences of these lengths over shuffled pages; -1 past a sequence's end."""
    n = [(l + PAGE - 1) // PAGE for l in lens]
    perm = (torch.randperm(max(1, sum(n)), generator=gen) + first_page).to(torch.int32)
    bt = torch.full((len(lens), max(1, max(n))), -1, dtype=torch.int32)
    at = 0
    for s, k in enumerate(n):
        bt[s, :k] = perm[at:at + k]
        at += k
    return bt.to(DEV), max(1, sum(n))


def _normal(shape, dtype, gen, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _inputs(case, seed):
    cpu, gpu = torch.Generator().manual_seed(seed), torch.Generator(DEV).manual_seed(seed)
    nkv, hd, dt = case["nkv"], case["hd"], DTYPES[case["dtype"]]
    ls = _lengths(case)
    if case["op"] == "evict":
        nl, ns, keep = case["layers"], len(ls), case["keep"]
        src, n_src = _table(ls, cpu)
        dst, n_dst = _table([min(l, keep) for l in ls], cpu, n_src)
        k = torch.empty((nl, n_src + n_dst, nkv, PAGE, hd), device=DEV, dtype=dt)
        v = torch.empty_like(k)
        for p in (k, v):
            for i in range(nl):
                p[i] = _normal(p[i].shape, dt, gpu)
        k[:, n_src:] = 0
        v[:, n_src:] = 0
        # accumulated weights: few keys hold most of the mass, many hold next
        # to none, and some were never seen at all (equal zeros)
        w = torch.exp(3.0 * torch.randn((nl, ns, nkv, max(ls)), generator=gpu, device=DEV) - 4.0)
        w = torch.where(w < 3e-4, torch.zeros_like(w), w)
        return {"case": case, "ls": ls, "k": k, "v": v, "src": src, "dst": dst, "n_src": n_src, "w": w,
                "kv_len": torch.tensor(ls, dtype=torch.int32, device=DEV),
                "kept": torch.full((nl, ns, nkv, keep), -1, dtype=torch.int32, device=DEV),
                "w_kept": torch.zeros((nl, ns, nkv, keep), device=DEV),
                "new_len": torch.zeros(ns, dtype=torch.int32, device=DEV)}
    nq = case["nq"]
    total = sum(n for n, _ in ls)
    bt, pages = _table([kv for _, kv in ls], cpu)
    k = _normal((pages, nkv, PAGE, hd), dt, gpu)
    v = _normal((pages, nkv, PAGE, hd), dt, gpu)
    # scores of a few units, as trained heads have: some rows attend to few keys
    q = _normal((total, nq, hd), dt, gpu, 2.0)
    starts = [0]
    for n, _ in ls:
        starts.append(starts[-1] + n)
    st = {"case": case, "ls": ls, "q": q, "k": k, "v": v, "bt": bt, "starts": starts,
          "q_start": torch.tensor(starts, dtype=torch.int32, device=DEV),
          "kv_len": torch.tensor([kv for _, kv in ls], dtype=torch.int32, device=DEV),
          "max_q": max(n for n, _ in ls), "max_kv": max(kv for _, kv in ls), "scale": 1.0 / math.sqrt(hd)}
    if case["op"] == "weights":
        st["lse"] = _attend_plain(st)[1]
        st["w_in"] = None if case["fresh"] else torch.exp(
            2.0 * torch.randn((len(ls), nkv, st["max_kv"]), generator=gpu, device=DEV) - 3.0)
        st["w_out"] = torch.zeros((len(ls), nkv, st["max_kv"]), device=DEV)
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if own:
        vv = _vvq2()
        st["pages"] = vv.Pages(st["k"], st["v"], st["src"] if case["op"] == "evict" else st["bt"])
    return st


# ------------------------------------------------------------ plain forms
def _blocks(st):
    """Groups of equally treated work: sequences with few rows as one padded
    batch, longer ones one by one in slices of rows."""
    ls = st["ls"]
    small = [s for s, (n, _) in enumerate(ls) if n <= 32]
    return small, [s for s, (n, _) in enumerate(ls) if n > 32]


def _gather(pool, bt, seqs, n_keys):
    """f32 [sequence][kv_head][key][hd] of the first n_keys keys."""
    pages = bt[seqs, :(n_keys + PAGE - 1) // PAGE].clamp(min=0).long()
    x = pool[pages]                                        # [s][page][kv][64][hd]
    s, p, g, _, hd = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(s, g, p * PAGE, hd)[:, :, :n_keys].float()


def _scores(st, q, k, lim):
    """q [s][t][nq][hd], k [s][g][j][hd], lim [s][t] -> masked scores [s][g][t*G][j]."""
    s, t, nq, hd = q.shape
    g = k.shape[1]
    x = q.float().reshape(s, t, g, nq // g, hd).transpose(1, 2).reshape(s, g, t * (nq // g), hd)
    x = torch.matmul(x, k.transpose(2, 3)) * st["scale"]
    lim = lim.repeat_interleave(nq // g, 1)[:, None, :, None]
    return x.masked_fill_(torch.arange(k.shape[2], device=DEV) >= lim, -math.inf)


def _steps(st):
    """(sequence ids, row ids [s][t], valid rows [s][t], q, key count, limits) of each block."""
    small, large = _blocks(st)
    ls, starts = st["ls"], st["starts"]
    if small:
        t = max(ls[s][0] for s in small)
        idx = torch.arange(t, device=DEV)[None, :]
        s = torch.tensor(small, device=DEV)
        n = (st["q_start"][s + 1] - st["q_start"][s])[:, None]
        ok = idx < n
        rows = torch.where(ok, st["q_start"][s][:, None] + idx, torch.zeros_like(idx)).long()
        lim = torch.where(ok, st["kv_len"][s][:, None] - n + idx + 1, torch.zeros_like(idx))
        yield s, rows, ok, st["q"][rows], max(ls[i][1] for i in small), lim
    for i in large:
        n, kv = ls[i]
        step = max(64, int(1.5e9 / 4 / (st["case"]["nq"] * kv)))
        for t0 in range(0, n, step):
            t1 = min(n, t0 + step)
            rows = torch.arange(starts[i] + t0, starts[i] + t1, device=DEV)[None, :]
            lim = torch.arange(kv - n + t0 + 1, kv - n + t1 + 1, device=DEV)[None, :]
            yield (torch.tensor([i], device=DEV), rows, torch.ones_like(rows, dtype=torch.bool), st["q"][rows],
                   kv - n + t1, lim)


def _rows_of(x, t):
    """[s][g][t*G][...] -> [s][t][g*G][...]"""
    s, g, r = x.shape[:3]
    return x.reshape(s, g, t, r // t, *x.shape[3:]).transpose(1, 2).reshape(s, t, g * (r // t), *x.shape[3:])


def _attend_plain(st):
    q = st["q"]
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], device=DEV)
    for s, rows, ok, qb, n_keys, lim in _steps(st):
        x = _scores(st, qb, _gather(st["k"], st["bt"], s, n_keys), lim)
        m = x.amax(-1, keepdim=True)
        m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
        p = x.sub_(m).exp_()
        z = p.sum(-1, keepdim=True)
        o = torch.matmul(p, _gather(st["v"], st["bt"], s, n_keys)) / torch.where(z > 0, z, torch.ones_like(z))
        t = rows.shape[1]
        out[rows[ok]] = _rows_of(o, t)[ok].to(q.dtype)
        lse[rows[ok]] = _rows_of((m + torch.log(z))[..., 0], t)[ok]
    return out, lse


def _weights_plain(st):
    w, w_in = st["w_out"], st["w_in"]
    acc = torch.zeros_like(w)
    for s, rows, ok, qb, n_keys, lim in _steps(st):
        t = rows.shape[1]
        x = _scores(st, qb, _gather(st["k"], st["bt"], s, n_keys), lim)
        l = st["lse"][rows]                                            # [s][t][nq]
        g, G = x.shape[1], l.shape[2] // x.shape[1]
        l = l.reshape(len(s), t, g, G).transpose(1, 2).reshape(len(s), g, t * G, 1)
        seen = (lim > 0).repeat_interleave(G, 1)[:, None, :, None]
        p = torch.where(seen, x - l, torch.full_like(x, -math.inf)).exp_()
        acc[s, :, :n_keys] += p.sum(2)
    j = torch.arange(w.shape[2], device=DEV)[None, None, :]
    kv = st["kv_len"][:, None, None]
    if w_in is not None:
        n = (st["q_start"][1:] - st["q_start"][:-1])[:, None, None]
        acc = torch.where(j < kv - n, acc + w_in, acc)
    w.copy_(torch.where(j < kv, acc, w))
    return w


def _evict_plain(st):
    c, w, kvl = st["case"], st["w"], st["kv_len"]
    nl, ns, nkv, width = w.shape
    keep = c["keep"]
    j = torch.arange(width, device=DEV)
    n = kvl[:, None]
    new_len = torch.clamp(kvl, max=keep)
    must = (j < c["first"]) | (j >= n - c["recent"])                    # [ns][width]
    rank = torch.where(must[None, :, None, :], torch.full_like(w, math.inf),
                       torch.where(torch.isnan(w), torch.full_like(w, -math.inf), w))
    # three groups, each in weight order: kept at any weight, the others, past the end
    group = torch.where(j >= n, 2, torch.where(must, 0, 1))[None, :, None, :].expand_as(w)
    by_w = torch.sort(rank, dim=-1, descending=True, stable=True)[1]
    by_g = torch.sort(torch.gather(group, -1, by_w), dim=-1, stable=True)[1]
    order = torch.gather(by_w, -1, by_g)[..., :keep]
    if order.shape[-1] < keep:
        order = torch.nn.functional.pad(order, (0, keep - order.shape[-1]))
    i = torch.arange(keep, device=DEV)
    ok = (i < new_len[:, None])[None, :, None, :].expand(nl, ns, nkv, keep)
    idx = torch.sort(torch.where(ok, order, torch.full_like(order, 1 << 40)), dim=-1)[0]
    idx = torch.where(ok, idx, torch.zeros_like(idx))
    st["kept"].copy_(torch.where(ok, idx, torch.full_like(idx, -1)))
    st["w_kept"].copy_(torch.where(ok, torch.gather(w, -1, idx), st["w_kept"]))
    st["new_len"].copy_(new_len)
    seq = torch.arange(ns, device=DEV)[:, None, None].expand(ns, nkv, keep)
    g = torch.arange(nkv, device=DEV)[None, :, None].expand(ns, nkv, keep)
    i = i[None, None, :].expand(ns, nkv, keep)
    for l in range(nl):
        okl = ok[l]
        sp = st["src"][seq, idx[l] // PAGE].long()[okl]
        dp = st["dst"][seq, (i // PAGE).clamp(max=st["dst"].shape[1] - 1)].long()[okl]
        at, to, gg = (idx[l] % PAGE)[okl], (i % PAGE)[okl], g[okl]
        for pool in (st["k"], st["v"]):
            pool[l][dp, gg, to] = pool[l][sp, gg, at]
    return _evicted(st)


def _evicted(st):
    n = st["n_src"]
    return {"kept": st["kept"], "new_len": st["new_len"], "w": st["w_kept"], "k": st["k"][:, n:], "v": st["v"][:, n:]}


def run(state):
    st, op = state, state["case"]["op"]
    if not own:
        if op == "attention":
            return _attend_plain(st)
        return _weights_plain(st) if op == "weights" else _evict_plain(st)
    vv = _vvq2()
    if op == "attention":
        return vv.attention_paged(st["q"], st["pages"], st["q_start"], st["kv_len"], st["max_q"], st["max_kv"],
                                  want_lse=True)
    if op == "weights":
        return vv.attention_key_weights(st["q"], st["lse"], st["pages"], st["q_start"], st["kv_len"], st["max_q"],
                                        st["max_kv"], w_in=st["w_in"], w_out=st["w_out"])
    c = st["case"]
    vv.pages_evict(st["pages"], st["dst"], st["kv_len"], st["w"], c["keep"], n_first=c["first"],
                   n_recent=c["recent"], kept=st["kept"], w_out=st["w_kept"], new_len=st["new_len"])
    return _evicted(st)


# ---------------------------------------------------------------- in 64 bits
def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "evict":
        return _evict_exact(st)
    nkv, hd, nq = case["nkv"], case["hd"], case["nq"]
    G = nq // nkv
    q, starts = st["q"], st["starts"]
    out = torch.zeros((q.shape[0], nq, hd), device=DEV, dtype=torch.float64)
    lse = torch.full((q.shape[0], nq), -math.inf, device=DEV, dtype=torch.float64)
    w = st["w_out"].double() if case["op"] == "weights" else None
    for s, (n, kv) in enumerate(st["ls"]):
        pages = st["bt"][s, :(kv + PAGE - 1) // PAGE].long()
        for g in range(nkv):
            K = st["k"][pages, g].reshape(-1, hd)[:kv].double()
            V = st["v"][pages, g].reshape(-1, hd)[:kv].double()
            if w is not None:
                w[s, g, :kv] = 0
            step = max(16, int(4e8 / 8 / (G * kv)))
            for t0 in range(0, n, step):
                t1 = min(n, t0 + step)
                see = kv - n + t1
                x = torch.einsum("thd,jd->thj", q[starts[s] + t0:starts[s] + t1, g * G:(g + 1) * G].double(), K[:see])
                x *= st["scale"]
                t = torch.arange(t0, t1, device=DEV)
                hidden = torch.arange(see, device=DEV)[None, :] > (kv - n + t)[:, None]
                x = x.masked_fill(hidden[:, None, :], -math.inf)
                if w is not None:
                    l = st["lse"][starts[s] + t0:starts[s] + t1, g * G:(g + 1) * G].double()
                    w[s, g, :see] += torch.exp(x - l[..., None]).sum((0, 1))
                    continue
                z = torch.logsumexp(x, -1)
                lse[starts[s] + t0:starts[s] + t1, g * G:(g + 1) * G] = z
                out[starts[s] + t0:starts[s] + t1, g * G:(g + 1) * G] = torch.exp(x - z[..., None]) @ V[:see]
            if w is not None and st["w_in"] is not None:
                w[s, g, :kv - n] += st["w_in"][s, g, :kv - n].double()
    return w if w is not None else (out, lse)


def _evict_exact(st):
    """Key by key on the host: the definition, without sorting tricks."""
    c = st["case"]
    if c["layers"] * c["nkv"] * sum(st["ls"]) > 4_000_000:
        return None
    keep, w = c["keep"], st["w"].double().cpu()
    for l in range(c["layers"]):
        for s, n in enumerate(st["ls"]):
            m = min(n, keep)
            for g in range(c["nkv"]):
                if n <= keep:
                    kept = list(range(n))
                else:
                    first, tail = min(c["first"], n), max(min(c["first"], n), n - c["recent"])
                    x = w[l, s, g, :n].tolist()
                    mid = sorted(range(first, tail), key=lambda j: (-x[j] if x[j] == x[j] else math.inf, j))
                    kept = sorted(list(range(first)) + list(range(tail, n)) + mid[:keep - first - (n - tail)])
                i = torch.arange(m, device=DEV)
                j = torch.tensor(kept, device=DEV)
                st["kept"][l, s, g, :m] = j.int()
                st["w_kept"][l, s, g, :m] = st["w"][l, s, g, j]
                sp, dp = st["src"][s, j // PAGE].long(), st["dst"][s, i // PAGE].long()
                for pool in (st["k"], st["v"]):
                    pool[l, dp, g, i % PAGE] = pool[l, sp, g, j % PAGE]
    st["new_len"].copy_(torch.clamp(st["kv_len"], max=keep))
    return _evicted(st)
