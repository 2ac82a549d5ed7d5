"""Timed cases of the paged-serving operators: the rotated append to a paged
K/V cache, decode attention over a shared prefix, and filtered sampling.

`run` computes an operator in its plain form (elementary torch operations), or
with `own` set through this package's kernels; `exact` restates each operator's
definition in 64 bits.  Head dim 128 and 16-row pages throughout, as the
package's paged cache has them.
"""
import math

import numpy as np
import torch

own = False

HD = 128
PAGE = 16
DEV = "cuda"


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of a full batch: 16 sequences, one token each
        dict(name="append decode 16", op="append", tokens=16, seqs=16, nh=16, nkv=2, kv="f16", prefix=512),
        # chunked prefill of a few prompts with decode rows among them, f32 cache
        dict(name="append mixed 1531 f32", op="append", tokens=1531, seqs=23, nh=28, nkv=4, kv="f32", prefix=0),
        # whole prompts of a batch in one pass, wide model
        dict(name="append prompts 16384", op="append", tokens=16384, seqs=8, nh=32, nkv=8, kv="f16", prefix=0),
        # two short chats over a short system prompt: latency
        dict(name="prefix 2x256", op="attn", seqs=2, pad=0, prefix=256, longest=32, nh=16, nkv=2, kv="f16"),
        # the package's batch of 16 in slots of 640 positions over a long system prompt
        dict(name="prefix 16x2048", op="attn", seqs=16, pad=0, prefix=2048, longest=640, nh=16, nkv=2, kv="f16"),
        # f32 cache, prefix and suffixes that end inside a page, a padded batch
        dict(name="prefix 17x1001 f32", op="attn", seqs=17, pad=3, prefix=1001, longest=333, nh=28, nkv=4, kv="f32"),
        # questions over one document: 64 sequences
        dict(name="prefix 64x8192", op="attn", seqs=64, pad=0, prefix=8192, longest=1024, nh=16, nkv=2, kv="f16"),
        # many samples of one long prompt
        dict(name="prefix 256x16384", op="attn", seqs=256, pad=0, prefix=16384, longest=512, nh=16, nkv=2, kv="f16"),
        # one stream, top-k 40: latency
        dict(name="sample 1 top-k", op="sample", rows=1, n=151936, k=40, p=1.0, minp=0.0, temp=0.8),
        # a batch of 16 with nucleus and min-p filters
        dict(name="sample 16 top-p min-p", op="sample", rows=16, n=151936, k=0, p=0.95, minp=0.02, temp=1.0),
        # an odd vocabulary, every filter
        dict(name="sample 7 of 5003", op="sample", rows=7, n=5003, k=200, p=0.9, minp=0.01, temp=1.3),
        # a large batch, no filter on some of its tail: mass over the whole row
        dict(name="sample 256 top-p", op="sample", rows=256, n=151936, k=0, p=0.98, minp=0.0, temp=1.1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    heads = [(16, 2), (16, 2), (28, 4), (32, 8), (8, 1), (4, 4)]
    op = rng.choice(["append", "attn", "attn", "sample"])
    nh, nkv = rng.choice(heads)
    kv = rng.choice(["f16", "f16", "f32"])
    if op == "append":
        tokens = _log_int(rng, 1, 16000)
        return dict(op=op, tokens=tokens, seqs=_log_int(rng, 1, min(tokens, 256)), nh=nh, nkv=nkv, kv=kv,
                    prefix=rng.choice([0, 1, 77, 512, 2000]))
    if op == "attn":
        seqs = _log_int(rng, 1, 250)
        cost = 4 if kv == "f32" else 1  # an f32 cache has twice the bytes and three products for each one
        prefix = rng.choice([0, 1]) if rng.random() < 0.1 else _log_int(
            rng, 2, max(2, min(16000, 256 * 16 * 16000 // (seqs * nh * cost))))
        longest = _log_int(rng, 1, max(1, min(4000, 256 * 2 * 500 // (seqs * nkv * cost))))
        return dict(op=op, seqs=seqs, pad=rng.choice([0, 0, 1, 5]), prefix=prefix, longest=longest, nh=nh, nkv=nkv, kv=kv)
    return dict(op="sample", rows=_log_int(rng, 1, 250), n=_log_int(rng, 64, 151936),
                k=rng.choice([0, 0, 1, 20, 64, 1000]), p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.99]),
                minp=rng.choice([0.0, 0.0, 0.05, 0.3]), temp=rng.choice([0.3, 0.7, 1.0, 1.0, 1.7]))


def _lens(c):
    """Suffix lengths, evenly spread from 0 to the longest (one sequence: the longest)."""
    n, m = c["seqs"], c["longest"]
    return [m] if n == 1 else [i * m // (n - 1) for i in range(n)]


def _runs(c):
    """Tokens of each sequence in an append: halving shares, one at least."""
    left, n = c["tokens"], c["seqs"]
    out = []
    for i in range(n):
        rest = n - 1 - i
        take = left if rest == 0 else max(1, min(left - rest, (left - rest) // 2 if c["tokens"] > 4 * n else left // (rest + 1)))
        out.append(take)
        left -= take
    return out


def work(c):
    if c["op"] == "append":
        esz = 2 if c["kv"] == "f16" else 4
        t, nh, nkv = c["tokens"], c["nh"], c["nkv"]
        longest = max(_runs(c))
        byt = t * (nh + 2 * nkv) * HD * 4 + t * nh * HD * 4 + 2 * t * nkv * HD * esz + t * 8 + longest * HD * 4
        return {"bytes": byt, "flops": t * (nh + nkv) * (HD // 2) * 6}
    if c["op"] == "attn":
        esz = 2 if c["kv"] == "f16" else 4
        keys = c["prefix"] + sum(_lens(c))
        byt = 2 * keys * c["nkv"] * HD * esz + 2 * c["seqs"] * c["nh"] * HD * 4 + keys // PAGE * 4
        return {"bytes": byt, "flops": 4 * HD * c["nh"] * (c["seqs"] * c["prefix"] + sum(_lens(c)))}
    return {"bytes": c["rows"] * (c["n"] * 4 + 32), "flops": c["rows"] * c["n"] * 4}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def _tables(n):
    """cos and sin of the rotation, [n][128], the second half a copy of the first (theta 1e6)."""
    inv = 1e6 ** (-torch.arange(0, HD, 2, dtype=torch.float64, device=DEV) / HD)
    a = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * inv[None, :]
    a = torch.cat([a, a], 1)
    return torch.cos(a).float().contiguous(), torch.sin(a).float().contiguous()


def prepare(case, seed):
    c = case
    g = _gen(seed)
    kv = torch.float16 if c.get("kv") == "f16" else torch.float32
    if c["op"] == "append":
        runs = _runs(c)
        first = [(i * 37) % 40 for i in range(c["seqs"])]  # rows a sequence holds already
        need = [(f + r + PAGE - 1) // PAGE for f, r in zip(first, runs)]
        total = sum(need) + 3
        perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        pages = torch.full((c["seqs"], max(need)), -1, dtype=torch.int32, device=DEV)
        ids = torch.split(perm[:sum(need)], need)
        for i, p in enumerate(ids):
            pages[i, :len(p)] = p
        slot = torch.cat([torch.full((r,), i, dtype=torch.int32) for i, r in enumerate(runs)])
        pos = torch.cat([torch.arange(f, f + r, dtype=torch.int32) for f, r in zip(first, runs)]) + c["prefix"]
        cos, sin = _tables(c["prefix"] + max(f + r for f, r in zip(first, runs)))
        w = (c["nh"] + 2 * c["nkv"]) * HD
        return dict(op="append", nh=c["nh"], prefix=c["prefix"], qkv=_randn(g, c["tokens"], w), slot=slot.to(DEV),
                    pos=pos.to(DEV), pages=pages, cos=cos, sin=sin,
                    kc=_randn(g, total, PAGE, c["nkv"], HD).to(kv), vc=_randn(g, total, PAGE, c["nkv"], HD).to(kv),
                    q_out=torch.zeros(c["tokens"], c["nh"] * HD, device=DEV))
    if c["op"] == "attn":
        lens = torch.tensor(_lens(c), dtype=torch.int32, device=DEV)
        lens = lens[torch.randperm(c["seqs"], generator=g, device=DEV)]
        lens = torch.cat([lens, torch.full((c["pad"],), -1, dtype=torch.int32, device=DEV)])  # padding of the batch
        n = c["seqs"] + c["pad"]
        np_, ns = (c["prefix"] + PAGE - 1) // PAGE, (c["longest"] + PAGE - 1) // PAGE
        total = np_ + n * ns
        perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
        return dict(op="attn", prefix=c["prefix"], longest=c["longest"], lens=lens, prefix_pages=perm[:np_].contiguous(),
                    pages=perm[np_:].reshape(n, ns).contiguous(), q=1.7 * _randn(g, n, c["nh"] * HD),
                    kc=_randn(g, total, PAGE, c["nkv"], HD, dtype=kv), vc=_randn(g, total, PAGE, c["nkv"], HD, dtype=kv),
                    out=torch.full((n, c["nh"] * HD), 0.25, device=DEV), err=torch.zeros(1, dtype=torch.int32, device=DEV))
    rows, n = c["rows"], c["n"]
    # a language model's next-token logits: a broad floor, some plausible tokens, every fourth row undecided
    logits = 2.0 * _randn(g, rows, n)
    m = min(40, n)
    at = torch.rand(rows, n, generator=g, device=DEV).topk(m).indices
    lift = 6.0 + 9.0 * torch.rand(rows, m, generator=g, device=DEV)
    lift[::4] = 2.0
    logits.scatter_(1, at, lift)
    full = lambda v, t: torch.full((rows,), v, dtype=t, device=DEV)  # noqa: E731
    return dict(op="sample", logits=logits, temp=full(c["temp"], torch.float32), k=full(c["k"], torch.int32),
                p=full(c["p"], torch.float32), minp=full(c["minp"], torch.float32),
                r=torch.rand(rows, generator=g, device=DEV), ids=torch.zeros(rows, dtype=torch.int32, device=DEV),
                probs=torch.zeros(rows, device=DEV))


# ---------------------------------------------------------------- plain forms
def _rotate(x, cos, sin):
    """x [T][heads][128], cos / sin [T][1][64]."""
    lo, hi = x[..., :HD // 2], x[..., HD // 2:]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _append_plain(s):
    nh, nkv = s["nh"], s["kc"].shape[2]
    t = s["qkv"].shape[0]
    x = s["qkv"].view(t, nh + 2 * nkv, HD)
    pos, slot = s["pos"].long(), s["slot"].long()
    cos, sin = s["cos"][pos][:, None, :HD // 2], s["sin"][pos][:, None, :HD // 2]
    at = pos - s["prefix"]
    row = s["pages"][slot, at // PAGE].long() * PAGE + at % PAGE
    s["kc"].view(-1, nkv, HD)[row] = _rotate(x[:, nh:nh + nkv], cos, sin).to(s["kc"].dtype)
    s["vc"].view(-1, nkv, HD)[row] = x[:, nh + nkv:].to(s["vc"].dtype)
    s["q_out"].copy_(_rotate(x[:, :nh], cos, sin).reshape(t, nh * HD))
    return s["q_out"], s["kc"], s["vc"]


def _attn_plain(s):
    n, nkv = s["q"].shape[0], s["kc"].shape[2]
    nh = s["q"].shape[1] // HD
    q = s["q"].view(n, nkv, nh // nkv, HD) * (1.0 / math.sqrt(HD))
    kc, vc = s["kc"].view(-1, nkv, HD), s["vc"].view(-1, nkv, HD)
    i = torch.arange(s["prefix"], device=DEV)
    prow = s["prefix_pages"][i // PAGE].long() * PAGE + i % PAGE
    j = torch.arange(s["longest"], device=DEV)
    srow = s["pages"][:, j // PAGE].long() * PAGE + j % PAGE
    live = (j[None, :] < s["lens"][:, None])[:, None, None, :]
    kp, vp = kc[prow].float(), vc[prow].float()
    ks, vs = kc[srow].float(), vc[srow].float()
    a = torch.einsum("bkgd,tkd->bkgt", q, kp)
    b = torch.einsum("bkgd,btkd->bkgt", q, ks).masked_fill(~live, -math.inf)
    sc = torch.cat([a, b], -1)
    top = sc.amax(-1, keepdim=True).clamp_min(-3e38)
    e = torch.exp(sc - top)
    z = e.sum(-1, keepdim=True)
    o = torch.einsum("bkgt,tkd->bkgd", e[..., :s["prefix"]], vp) + torch.einsum("bkgt,btkd->bkgd", e[..., s["prefix"]:], vs)
    o = torch.where(z > 0, o / z.clamp_min(1e-30), torch.zeros_like(o)).reshape(n, nh * HD)
    return torch.where((s["lens"] < 0)[:, None], s["out"], o)


def _sample_plain(s):
    x = s["logits"].masked_fill(~(s["logits"] >= -1e30), -math.inf)  # NaN and masked tokens are never taken
    v, ix = torch.sort(x, dim=1, descending=True, stable=True)
    n = x.shape[1]
    rank = torch.arange(n, device=DEV)[None, :]
    t = torch.where(s["temp"] > 0, s["temp"], torch.ones_like(s["temp"])).double()[:, None]
    w = torch.exp((v.double() - v[:, :1].double()) / t)
    k = torch.where(s["k"] > 0, s["k"], torch.full_like(s["k"], n))[:, None]
    w = w.masked_fill(rank >= k, 0.0)
    cum = torch.cumsum(w, 1)
    p, minp = s["p"].double()[:, None], s["minp"].double()[:, None]
    keep = (rank < k) & ((p >= 1) | (cum - w < p * cum[:, -1:])) & (w >= minp)
    keep[:, 0] = True
    last = keep.sum(1, keepdim=True) - 1
    mass = cum.gather(1, last)
    at = (cum < s["r"].double()[:, None] * mass).sum(1, keepdim=True).minimum(last)
    return ix.gather(1, at)[:, 0].to(torch.int32), (w.gather(1, at) / mass)[:, 0].float()


# ---------------------------------------------------------------- one pass
def run(state):
    s = state
    if not own:
        return {"append": _append_plain, "attn": _attn_plain, "sample": _sample_plain}[s["op"]](s)
    from vibethinker_webgpu_lora_b200 import kernels as K
    if s["op"] == "append":
        K.kv_append_paged(s["qkv"], s["pos"], s["slot"], s["pages"], s["kc"], s["vc"], s["cos"], s["sin"], s["nh"],
                          q_out=s["q_out"], prefix_len=s["prefix"])
        return s["q_out"], s["kc"], s["vc"]
    if s["op"] == "attn":
        if "ws" not in s:  # the workspace is the caller's and is kept
            nh, nkv = s["q"].shape[1] // HD, s["kc"].shape[2]
            s["ws"] = torch.empty(K.attn_shared_prefix_bytes(s["q"].shape[0], nh, nkv, s["prefix"], s["longest"]),
                                  dtype=torch.uint8, device=DEV)
        K.attn_shared_prefix(s["q"], s["kc"], s["vc"], s["prefix_pages"], s["prefix"], s["pages"], s["lens"],
                             s["longest"], s["out"], s["ws"], err=s["err"])
        return s["out"]
    K.sample_filtered(s["logits"], s["r"], s["ids"], temp=s["temp"], top_k=s["k"], top_p=s["p"], min_p=s["minp"],
                      probs=s["probs"])
    return s["ids"], s["probs"]


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "append":
        return _append_exact(s)
    return _attn_exact(s) if s["op"] == "attn" else _sample_exact(s)


def _append_exact(s):
    """A token's pair (x_i, x_{i+64}) turned by its position's angle, as a complex product."""
    nh, nkv = s["nh"], s["kc"].shape[2]
    x = s["qkv"].double().reshape(-1, nh + 2 * nkv, 2, HD // 2)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long(), :HD // 2]
    z = torch.complex(x[:, :, 0], x[:, :, 1]) * turn[:, None]
    z = torch.cat([z.real, z.imag], -1)
    x = x.reshape(-1, nh + 2 * nkv, HD)
    kc, vc = s["kc"].double(), s["vc"].double()
    at = s["pos"].long() - s["prefix"]
    page = s["pages"].long()[s["slot"].long(), torch.div(at, PAGE, rounding_mode="floor")]
    kc[page, at % PAGE] = z[:, nh:nh + nkv]
    vc[page, at % PAGE] = x[:, nh + nkv:]
    return z[:, :nh].reshape(-1, nh * HD), kc, vc


def _attn_exact(s):
    """Each sequence by itself over its own keys: the prefix, then its suffix."""
    n, nkv = s["q"].shape[0], s["kc"].shape[2]
    nh = s["q"].shape[1] // HD
    out = s["out"].double()

    def rows(pages, count, pool):
        got = pool[pages[:(count + PAGE - 1) // PAGE].long()].reshape(-1, nkv, HD)
        return got[:count].double()

    kp, vp = (rows(s["prefix_pages"], s["prefix"], s[c]) for c in ("kc", "vc"))
    for b, m in enumerate(s["lens"].tolist()):
        if m < 0:
            continue
        k = torch.cat([kp, rows(s["pages"][b], m, s["kc"])])
        v = torch.cat([vp, rows(s["pages"][b], m, s["vc"])])
        if not len(k):
            out[b] = 0
            continue
        q = s["q"][b].double().view(nkv, nh // nkv, HD)
        p = torch.softmax(torch.matmul(q, k.permute(1, 2, 0)) / math.sqrt(HD), -1)
        out[b] = torch.matmul(p, v.permute(1, 0, 2)).reshape(-1)
    return out


def _sample_exact(s):
    """Row by row: the tokens in falling order, cut by each filter, then the first whose share reaches r."""
    x = s["logits"].cpu().numpy().astype(np.float64)
    par = [s[k].cpu().numpy().astype(np.float64) for k in ("temp", "k", "p", "minp", "r")]
    ids, probs = np.zeros(len(x), np.int32), np.zeros(len(x))
    for i, (row, t, k, p, minp, r) in enumerate(zip(x, *par)):
        order = np.argsort(-row, kind="stable")
        order = order[:int(k)] if k > 0 else order
        w = np.exp((row[order] - row[order[0]]) / t)
        n = len(w)
        if p < 1:
            n = min(n, int(np.searchsorted(np.cumsum(w), p * w.sum())) + 1)
        n = min(n, max(1, int((w >= minp).sum())))
        c = np.cumsum(w[:n])
        j = min(int(np.searchsorted(c, r * c[-1])), n - 1)
        ids[i], probs[i] = order[j], w[j] / c[-1]
    return torch.from_numpy(ids), torch.from_numpy(probs)
