"""The operators over cached sequences (afterimage_b200.runtime.seq_ops) as
cases to measure: attention of whole packed prompts, attention of a drafted
tree over a cache, the rotary embedding and cache write in front of both, and
the cache rows kept after a draft was accepted.

`run` computes an operator in plain torch (fp32 inside, one rounding at the
end) or, when `own` is set, through the package. Heads, head sizes and layer
counts are those of the benchmark's models (bench.py) or a rank's share of
them; a head size of 64 is generic.
"""
import math

import torch

own = False

BF16 = torch.bfloat16
DEV = "cuda"


# -- cases ---------------------------------------------------------------------
def listed():
    return [
        # one long prompt on the 14B shape: the compute-bound end
        dict(name="prompt-one-long", op="prompt", nh=40, nkv=8, hd=128, lens="16384", ctx="", max_len=0),
        # prompts of very different lengths packed into one pass (8B shape)
        dict(name="prompt-packed-ragged", op="prompt", nh=32, nkv=8, hd=128, lens="1,7,37,129,513,1000,2047,4099",
             ctx="", max_len=0),
        # many chat-sized prompts in one pass (0.6B shape): latency and row use count
        dict(name="prompt-short-batch", op="prompt", nh=16, nkv=8, hd=128,
             lens="17,64,33,96,5,71,48,88,23,64,19,52,90,41,77,12,64,35,81,58,29,67,93,44,14,60,38,85,50,26,73,9",
             ctx="", max_len=0),
        # the next piece of two long prompts, over what their caches hold already, on one of 8 ranks of
        # the 14B shape: few rows, long axis
        dict(name="prompt-over-cache", op="prompt", nh=5, nkv=1, hd=128, lens="256,61", ctx="7744,4039",
             max_len=8192),
        # a single token on the 14B shape: the smallest call of a generation loop
        dict(name="tree-one-token", op="tree", nh=40, nkv=8, hd=128, pos="1000", parents="-1", max_len=1152),
        # the pending token and four proposals in a chain, as draft/target speculation verifies them (8B shape)
        dict(name="tree-chain", op="tree", nh=32, nkv=8, hd=128, pos="4099", parents="-1,0,1,2,3", max_len=8192),
        # a wide tree over a long cache (14B shape): bytes and matrix work are both large
        dict(name="tree-wide-long", op="tree", nh=40, nkv=8, hd=128, pos="32000",
             parents="-1,0,0,0,0,0,0,0,1,1,1,1,2,2,2,3,3,3,4,4,5,5,6,7,8,8,8,9,9,10,12,12,13,15,15,18,24,24,24,25,25,"
                     "27,30,30,33,36,36,37,39,41,42,45,45,46,48,49,51,51,52,53,55,57,58,60", max_len=32768),
        # sixteen sequences, each with the same 26-node tree at a place of its own, heads of 64
        dict(name="tree-batch", op="tree", nh=32, nkv=8, hd=64,
             pos="4000,17,1311,2900,640,3777,95,2048,3333,1000,511,3900,2222,1,3001,768",
             parents="-1,0,0,0,0,1,1,1,2,2,3,3,4,5,5,6,8,8,10,13,13,14,16,19,19,21", max_len=4096),
        # a drafted tree's rotary embedding and cache write, far into a cache (14B shape, q/k norms)
        dict(name="rope-draft-tree", op="rope", nh=40, nkv=8, hd=128, lens="26", start="20011",
             parents="-1,0,0,0,0,1,1,1,2,2,3,3,4,5,5,6,8,8,10,13,13,14,16,19,19,21", norm=True, theta=1e6,
             max_len=20480),
        # three packed prompts, 8192 tokens together (8B shape, no norms)
        dict(name="rope-prompts", op="rope", nh=32, nkv=8, hd=128, lens="5000,3001,191", start="0,130,7",
             parents="", norm=False, theta=5e5, max_len=5120),
        # an accepted path of five in all 40 layers of one sequence (14B shape)
        dict(name="keep-one", op="keep", layers=40, nkv=8, hd=128, pos="611", keep="0,5,9,17,40", max_len=1024),
        # sixteen sequences, 32 layers, paths of different lengths (-1: the row stays)
        dict(name="keep-batch", op="keep", layers=32, nkv=8, hd=128,
             pos="100,17,311,290,64,377,95,204,333,10,51,390,222,1,301,68",
             keep="0,8,11,15,19,-1,-1,-1;0,9,-1,-1,-1,-1,-1,-1;0,8,12,18,21,23,24,25;0,-1,-1,-1,-1,-1,-1,-1;"
                  "0,10,12,-1,-1,-1,-1,-1;0,8,13,20,-1,-1,-1,-1;0,9,14,-1,-1,-1,-1,-1;0,-1,-1,-1,-1,-1,-1,-1;"
                  "0,8,11,15,19,22,-1,-1;0,9,-1,-1,-1,-1,-1,-1;0,10,13,18,21,-1,-1,-1;0,8,-1,-1,-1,-1,-1,-1;"
                  "0,9,12,-1,-1,-1,-1,-1;0,8,13,20,-1,-1,-1,-1;0,9,14,-1,-1,-1,-1,-1;0,11,-1,-1,-1,-1,-1,-1",
             max_len=512),
    ]


HEADS = ((40, 8, 128), (32, 8, 128), (16, 8, 128), (5, 1, 128), (4, 1, 128), (20, 4, 128), (32, 8, 64), (8, 8, 64))


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _text(v):
    return ",".join(str(int(x)) for x in v)


def _tree(rng, n):
    """Parents of a random tree in topological order, the first node its root."""
    return [-1] + [rng.randrange(max(0, (i - 1) // 4), i) for i in range(1, n)]


def draw(rng):
    nh, nkv, hd = rng.choice(HEADS)
    op = rng.choice(("prompt", "prompt", "tree", "tree", "rope", "keep"))
    if op == "prompt":
        if rng.random() < 0.3:  # over caches
            b = rng.randint(1, 4)
            lens = [_log(rng, 1, 1024) for _ in range(b)]
            ctx = [rng.randint(0, 12000) for _ in range(b)]
            top = max(a + c for a, c in zip(lens, ctx))
            return dict(op=op, nh=nh, nkv=nkv, hd=hd, lens=_text(lens), ctx=_text(ctx), max_len=top + rng.randint(0, 500))
        total = _log(rng, 16, 12000)
        lens = []
        while sum(lens) < total and len(lens) < 64:
            lens.append(min(_log(rng, 1, total), total - sum(lens)))
        return dict(op=op, nh=nh, nkv=nkv, hd=hd, lens=_text(lens), ctx="", max_len=0)
    if op == "tree":
        b = rng.choice((1, 1, 1, 2, 5, 16))
        top = _log(rng, 1, 40000 // b)
        pos = [top] + [rng.randint(0, top) for _ in range(b - 1)]
        n = _log(rng, 1, 96)
        return dict(op=op, nh=nh, nkv=nkv, hd=hd, pos=_text(pos), parents=_text(_tree(rng, n)),
                    max_len=top + n + rng.randint(0, 300))
    if op == "rope":
        if rng.random() < 0.5:
            n, b = _log(rng, 1, 96), rng.choice((1, 2, 7))
            lens, parents = [n] * b, _text(_tree(rng, n))
        else:
            b = rng.randint(1, 8)
            lens, parents = [_log(rng, 1, 8192 // b) for _ in range(b)], ""
        start = [rng.randint(0, 6000) for _ in range(b)]
        return dict(op=op, nh=nh, nkv=nkv, hd=hd, lens=_text(lens), start=_text(start), parents=parents,
                    norm=rng.random() < 0.5, theta=rng.choice((5e5, 1e6)),
                    max_len=max(a + s for a, s in zip(lens, start)) + rng.randint(0, 100))
    b, n = rng.choice((1, 2, 6)), rng.randint(1, 12)
    keep = []
    for _ in range(b):
        m = rng.randint(1, n)
        path = sorted(rng.sample(range(n, n + 64), m - 1))  # a place is either kept where it is or comes from behind the path
        keep.append([0] + path + [-1] * (n - m))
    pos = [rng.randint(0, 400) for _ in range(b)]
    return dict(op=op, layers=rng.choice((28, 32, 40)), nkv=nkv, hd=hd, pos=_text(pos),
                keep=";".join(_text(k) for k in keep), max_len=max(pos) + n + 64 + rng.randint(0, 99))


# -- inputs --------------------------------------------------------------------
def _ints(text):
    return [int(x) for x in text.split(",")] if text else []


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _visible(parents):
    """bool [T, T]: a node sees itself and its ancestors."""
    n = len(parents)
    m = torch.zeros(n, n, dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            m[i] = m[p]
        m[i, i] = True
    return m


def _depths(parents):
    d = []
    for p in parents:
        d.append(d[p] + 1 if p >= 0 else 0)
    return d


def _long(v):
    return torch.tensor(v, dtype=torch.int64, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * by).to(BF16)

    op, nkv, hd = case["op"], case["nkv"], case["hd"]
    s = dict(op=op, case=case)
    if op == "prompt":
        # queries and keys of size 1 to 1.5 a value, as after q/k norms: scores with a spread of about 1.5
        nh, lens, ctx = case["nh"], _ints(case["lens"]), _ints(case["ctx"])
        s.update(q=normal(sum(lens), nh, hd, by=1.5), scale=hd ** -0.5, lens=lens, ctx=ctx, cu=_long(_cu(lens)))
        if ctx:
            s.update(k=normal(len(lens), nkv, case["max_len"], hd), v=normal(len(lens), nkv, case["max_len"], hd),
                     len_k=_long([a + c for a, c in zip(lens, ctx)]))
        else:
            s.update(k=normal(sum(lens), nkv, hd), v=normal(sum(lens), nkv, hd))
    elif op == "tree":
        nh, pos, parents = case["nh"], _ints(case["pos"]), _ints(case["parents"])
        b, t = len(pos), len(parents)
        s.update(q=normal(b, t, nh, hd, by=1.5), k=normal(b, nkv, case["max_len"], hd),
                 v=normal(b, nkv, case["max_len"], hd), pos=_long(pos), mask=_visible(parents).to(DEV),
                 top=max(pos) + t, scale=hd ** -0.5)
    elif op == "rope":
        nh, lens, start, parents = case["nh"], _ints(case["lens"]), _ints(case["start"]), _ints(case["parents"])
        n, b = sum(lens), len(lens)
        s.update(qkv=normal(n, (nh + 2 * nkv) * hd), cu=_long(_cu(lens)), start=_long(start),
                 depth=_long(_depths(parents) * b) if parents else None,
                 inv_freq=1.0 / (case["theta"] ** (torch.arange(0, hd, 2, device=DEV, dtype=torch.float32) / hd)),
                 q_norm=(1 + 0.2 * torch.randn(hd, device=DEV, generator=g)).to(BF16) if case["norm"] else None,
                 k_norm=(1 + 0.2 * torch.randn(hd, device=DEV, generator=g)).to(BF16) if case["norm"] else None,
                 k=torch.zeros(b, nkv, case["max_len"], hd, device=DEV, dtype=BF16),
                 v=torch.zeros(b, nkv, case["max_len"], hd, device=DEV, dtype=BF16))
    else:
        pos, keep = _ints(case["pos"]), [_ints(k) for k in case["keep"].split(";")]
        s.update(caches=normal(2 * case["layers"], len(pos), nkv, case["max_len"], hd), pos=_long(pos),
                 keep=_long(keep))
        s["list"] = list(s["caches"].unbind(0))  # one tensor a layer for keys and for values, as a program holds them
    return s


# -- the operators ---------------------------------------------------------------
def _softmax_values(scores, seen, v):
    """Rows of softmax(scores where seen) times v; a row that sees nothing is zero."""
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    return p.matmul(v) / total.clamp_min(1e-30)


def _plain_prompt(s):
    """Every prompt in turn, 1024 queries at a time against the keys that they may see."""
    q, nkv, ctx = s["q"], s["case"]["nkv"], s["ctx"]
    n, nh, hd = q.shape
    out = torch.empty_like(q)
    at = 0
    for i, m in enumerate(s["lens"]):
        c = ctx[i] if ctx else 0
        k = s["k"][i].float() if ctx else s["k"][at:at + m].float().transpose(0, 1)
        v = s["v"][i].float() if ctx else s["v"][at:at + m].float().transpose(0, 1)
        for lo in range(0, m, 1024):
            hi = min(m, lo + 1024)
            qq = q[at + lo:at + hi].float().reshape(hi - lo, nkv, nh // nkv, hd).permute(1, 2, 0, 3)
            qq = qq.reshape(nkv, -1, hd)
            scores = qq.matmul(k[:, :c + hi].transpose(1, 2)) * s["scale"]
            seen = torch.arange(c + hi, device=DEV) <= c + torch.arange(lo, hi, device=DEV)[:, None]
            o = _softmax_values(scores, seen.repeat(nh // nkv, 1), v[:, :c + hi])
            out[at + lo:at + hi] = o.reshape(nkv, nh // nkv, hi - lo, hd).permute(2, 0, 1, 3).reshape(hi - lo, nh, hd)
        at += m
    return out


def _plain_tree(s):
    q, top, mask, pos = s["q"], s["top"], s["mask"], s["pos"]
    b, t, nh, hd = q.shape
    nkv = s["k"].shape[1]
    k, v = s["k"][:, :, :top].float(), s["v"][:, :, :top].float()
    qq = q.float().reshape(b, t, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(b, nkv, -1, hd)
    scores = qq.matmul(k.transpose(2, 3)) * s["scale"]
    col = torch.arange(top, device=DEV) - pos[:, None]                      # [b, top]: the drafted node at a slot
    node = mask[:, col.clamp(0, t - 1)].permute(1, 0, 2) & (col < t)[:, None]  # [b, t, top]
    seen = node | (col < 0)[:, None]
    o = _softmax_values(scores, seen[:, None].repeat(1, 1, nh // nkv, 1), v)
    return o.reshape(b, nkv, nh // nkv, t, hd).permute(0, 3, 1, 2, 4).reshape(b, t, nh, hd).to(BF16)


def _plain_rope(s):
    nh, nkv, hd, eps = s["case"]["nh"], s["case"]["nkv"], s["case"]["hd"], 1e-6
    n = s["qkv"].shape[0]
    x = s["qkv"].float().reshape(n, nh + 2 * nkv, hd)
    seq = torch.searchsorted(s["cu"], torch.arange(n, device=DEV), right=True) - 1
    at = torch.arange(n, device=DEV) - s["cu"][seq]
    slot = s["start"][seq] + at
    place = s["start"][seq] + (at if s["depth"] is None else s["depth"])
    angle = place.double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float().repeat(1, 2)[:, None], angle.sin().float().repeat(1, 2)[:, None]

    def turn(h, w):
        if w is not None:
            h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * w.float()
        half = hd // 2
        return h * cos + torch.cat((-h[..., half:], h[..., :half]), -1) * sin

    s["k"][seq, :, slot] = turn(x[:, nh:nh + nkv], s["k_norm"]).to(BF16)
    s["v"][seq, :, slot] = x[:, nh + nkv:].to(BF16)
    return turn(x[:, :nh], s["q_norm"]).to(BF16), s["k"], s["v"]


def _plain_keep(s):
    caches, pos, keep = s["caches"], s["pos"], s["keep"]
    b, n = keep.shape
    place = torch.arange(n, device=DEV)
    src = pos[:, None] + torch.where(keep >= 0, keep, place)
    dst = pos[:, None] + place
    row = torch.arange(b, device=DEV)[:, None]
    caches[:, row, :, dst] = caches[:, row, :, src]
    return caches


def _own(s):
    from afterimage_b200.runtime import seq_ops
    if s["op"] == "prompt":
        return seq_ops.prompt_attention(s["q"], s["k"], s["v"], s["cu"], s["scale"], len_k=s.get("len_k"))
    if s["op"] == "tree":
        return seq_ops.tree_attention(s["q"], s["k"], s["v"], s["pos"], s["mask"], s["scale"])
    if s["op"] == "rope":
        c = s["case"]
        q = seq_ops.rope_cache_packed(s["qkv"], c["nh"], c["nkv"], c["hd"], s["cu"], s["start"], s["inv_freq"], s["k"],
                                      s["v"], depth=s["depth"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6)
        return q, s["k"], s["v"]
    seq_ops.keep_cache_rows(s["list"], s["pos"], s["keep"])
    return s["caches"]


def run(state):
    if own:
        return _own(state)
    return {"prompt": _plain_prompt, "tree": _plain_tree, "rope": _plain_rope, "keep": _plain_keep}[state["op"]](state)


# -- what a pass cannot do without -------------------------------------------------
def work(case):
    op, nkv, hd = case["op"], case["nkv"], case["hd"]
    if op == "prompt":
        nh, lens, ctx = case["nh"], _ints(case["lens"]), _ints(case["ctx"])
        ctx = ctx or [0] * len(lens)
        pairs = sum(m * c + m * (m + 1) // 2 for m, c in zip(lens, ctx))
        rows = 2 * sum(lens) * nh + 2 * sum(m + c for m, c in zip(lens, ctx)) * nkv
        return {"bytes": 2 * hd * rows, "flops": 4 * hd * nh * pairs}
    if op == "tree":
        nh, pos, parents = case["nh"], _ints(case["pos"]), _ints(case["parents"])
        t = len(parents)
        nodes = int(_visible(parents).sum())
        rows = 2 * len(pos) * t * nh + 2 * sum(p + t for p in pos) * nkv
        return {"bytes": 2 * hd * rows + t * t, "flops": 4 * hd * nh * sum(p * t + nodes for p in pos)}
    if op == "rope":
        n, heads = sum(_ints(case["lens"])), case["nh"] + 2 * nkv
        return {"bytes": 4 * n * heads * hd, "flops": n * heads * hd * (7 if case["norm"] else 3)}
    moved = sum(k >= 0 and k != i for row in case["keep"].split(";") for i, k in enumerate(_ints(row)))
    return {"bytes": 2 * 2 * 2 * case["layers"] * nkv * hd * moved, "flops": 0}


# -- the same in 64 bits, from the definitions ---------------------------------------
def _attend(q, k, v, seen, scale):
    """One head in 64 bits: q [t, hd], k and v [l, hd], seen bool [t, l]."""
    z = torch.einsum("td,ld->tl", q.double(), k.double()) * scale
    z = torch.where(seen, z, torch.full_like(z, -math.inf))
    w = torch.nan_to_num(torch.softmax(z, -1), nan=0.0)  # a row that sees nothing: no weights
    return torch.einsum("tl,ld->td", w, v.double())


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "keep":
        return None  # rows are copied, not computed: the plain form's are the bits themselves
    if op == "prompt":
        nh, group = case["nh"], case["nh"] // case["nkv"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        bounds = _cu(s["lens"])
        for i, m in enumerate(s["lens"]):
            rows = slice(bounds[i], bounds[i + 1])
            c = s["ctx"][i] if s["ctx"] else 0
            key = torch.arange(c + m, device=DEV)
            for h in range(nh):
                k = s["k"][i, h // group, :c + m] if s["ctx"] else s["k"][rows, h // group]
                v = s["v"][i, h // group, :c + m] if s["ctx"] else s["v"][rows, h // group]
                for part in range(0, m, 4096):
                    t = torch.arange(part, min(m, part + 4096), device=DEV)
                    out[bounds[i] + t, h] = _attend(s["q"][bounds[i] + t, h], k, v, key[None] <= (c + t)[:, None],
                                                    s["scale"])
        return out
    if op == "tree":
        nh, group, pos = case["nh"], case["nh"] // case["nkv"], _ints(case["pos"])
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        for i, p in enumerate(pos):
            t = s["mask"].shape[0]
            seen = torch.cat((torch.ones(t, p, dtype=torch.bool, device=DEV), s["mask"]), 1)
            for h in range(nh):
                out[i, :, h] = _attend(s["q"][i, :, h], s["k"][i, h // group, :p + t], s["v"][i, h // group, :p + t],
                                       seen, s["scale"])
        return out
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    n = s["qkv"].shape[0]
    x = s["qkv"].double().view(n, nh + 2 * nkv, hd)
    kc, vc = s["k"].double(), s["v"].double()
    q = torch.empty(n, nh, hd, dtype=torch.float64, device=DEV)
    bounds, starts = _cu(_ints(case["lens"])), _ints(case["start"])
    freq = torch.cat((s["inv_freq"], s["inv_freq"])).double()
    sign = torch.ones(hd, dtype=torch.float64, device=DEV)
    sign[:hd // 2] = -1
    for i, p in enumerate(starts):
        lo, hi = bounds[i], bounds[i + 1]
        step = torch.arange(hi - lo, device=DEV) if s["depth"] is None else s["depth"][lo:hi]
        a = (p + step).double()[:, None, None] * freq

        def rotated(h, w):
            if w is not None:
                h = w.double() * h / torch.sqrt((h * h).sum(-1, keepdim=True) / hd + 1e-6)
            return h * torch.cos(a) + sign * h.roll(hd // 2, -1) * torch.sin(a)

        q[lo:hi] = rotated(x[lo:hi, :nh], s["q_norm"])
        kc[i, :, p:p + hi - lo] = rotated(x[lo:hi, nh:nh + nkv], s["k_norm"]).transpose(0, 1)
        vc[i, :, p:p + hi - lo] = x[lo:hi, nh + nkv:].transpose(0, 1)
    return q, kc, vc
