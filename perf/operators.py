"""Cases of the training operators: attention, layer norm and token embedding, each with its backward pass.

`run` with `own` false computes them with elementary torch operations in 32 bits; with `own` true through diffbir_amd.ops."""
import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
D = 64   # head dimension of every attention of this framework


def listed():
    return [
        # the text tower's causal attention for a pair of prompts: latency
        dict(name="attn_text", op="attention", dir="step", dtype="f16", B=2, H=16, Hkv=16, Lq=77, Lk=77, causal=True, ragged=False),
        # self-attention of the 64x64 latent level at batch 8: the largest
        dict(name="attn_self_64", op="attention", dir="step", dtype="f16", B=8, H=5, Hkv=5, Lq=4096, Lk=4096, causal=False, ragged=False),
        # the same level attending to the prompt: few keys, many queries
        dict(name="attn_cross_64", op="attention", dir="step", dtype="bf16", B=8, H=5, Hkv=5, Lq=4096, Lk=77, causal=False, ragged=False),
        # self-attention of the 16x16 level: many heads, short rows
        dict(name="attn_self_16", op="attention", dir="step", dtype="bf16", B=8, H=20, Hkv=20, Lq=256, Lk=256, causal=False, ragged=False),
        # a padded batch of texts of unlike lengths, key / value heads shared by four
        dict(name="attn_padded", op="attention", dir="step", dtype="bf16", B=4, H=8, Hkv=2, Lq=1025, Lk=1025, causal=True, ragged=True),
        # one token over a long context
        dict(name="attn_token", op="attention", dir="fwd", dtype="f16", B=2, H=10, Hkv=10, Lq=1, Lk=9001, causal=False, ragged=False),
        # the text tower's norm on its 32-bit stream: latency
        dict(name="ln_text", op="layernorm", dir="step", dtype="f32", rows=154, C=1024, res=False),
        # a transformer block's norm at the 64x64 level, batch 8, with the residual's gradient
        dict(name="ln_block_64", op="layernorm", dir="step", dtype="f16", rows=32768, C=320, res=True),
        # an odd width: rows that no wide load is aligned to
        dict(name="ln_odd", op="layernorm", dir="step", dtype="bf16", rows=4099, C=1283, res=True),
        # a pair of prompts through the text tower's table: the gradient is nearly all zeros
        dict(name="emb_text", op="embedding", dir="step", table="f32", dtype="f32", B=2, L=77, V=49408, W=1024, pos=True, pad=0.8),
        # a large batch of prompts, mostly padding
        dict(name="emb_batch", op="embedding", dir="step", table="f32", dtype="bf16", B=512, L=77, V=49408, W=1024, pos=True, pad=0.7),
        # a small table of odd width in 16 bits
        dict(name="emb_odd", op="embedding", dir="step", table="bf16", dtype="bf16", B=3, L=1001, V=1009, W=333, pos=False, pad=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["attention", "attention", "layernorm", "embedding"])
    way = rng.choice(["fwd", "step", "step"])
    if op == "attention":
        H = rng.choice([1, 2, 4, 5, 8, 10, 20])
        Hkv = rng.choice([h for h in (1, 2, 4, 5, 8, 10, 20) if H % h == 0])
        B, Lq = rng.randint(1, 8), _log(rng, 1, 4096)
        Lk = max(2 if way == "step" else 1, rng.choice([Lq, _log(rng, 1, 300), _log(rng, 1, 9216)]))   # one key has no gradient through its score
        while B * H * Lq * Lk > 8 * 5 * 4096 * 4096:
            if B > 1:
                B -= 1
            else:
                Lk = Lk // 2
        return dict(op=op, dir=way, dtype=rng.choice(["f16", "bf16"]), B=B, H=H, Hkv=Hkv, Lq=Lq, Lk=Lk,
                    causal=rng.random() < 0.4, ragged=rng.random() < 0.3)
    if op == "layernorm":
        C = rng.choice([320, 640, 1280, 1024, _log(rng, 8, 8192), _log(rng, 1, 1024) * 8])
        rows = min(_log(rng, 1, 65536), 80_000_000 // C)
        return dict(op=op, dir=way, dtype=rng.choice(["f16", "bf16", "f32"]), rows=rows, C=C, res=rng.random() < 0.5)
    W = rng.choice([1024, 768, _log(rng, 1, 1024), _log(rng, 8, 256) * 8])
    V = rng.choice([49408, _log(rng, 2, 65536)])
    L = rng.choice([77, _log(rng, 1, 4096)])
    B = max(1, min(_log(rng, 1, 1024), 40000 // L))
    V = min(V, 60_000_000 // W)
    return dict(op=op, dir=way, table=rng.choice(["f32", "bf16", "f16"]), dtype=rng.choice(["f32", "bf16", "f16"]), B=B, L=L, V=V, W=W,
                pos=rng.random() < 0.5, pad=rng.choice([0.0, 0.3, 0.8]))


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    if c["op"] == "attention":
        t, B = _DT[c["dtype"]], c["B"]
        st = dict(case=c, q=(1.5 * randn(B, c["Lq"], c["H"], D)).to(t), k=randn(B, c["Lk"], c["Hkv"], D).to(t),
                  v=randn(B, c["Lk"], c["Hkv"], D).to(t), dout=(0.1 * randn(B, c["Lq"], c["H"], D)).to(t), q_len=None, kv_len=None)
        if c["ragged"]:   # samples of unlike lengths; a padded text has as many queries as keys
            st["kv_len"] = torch.randint(0, c["Lk"] + 1, (B,), device="cuda", generator=g, dtype=torch.int32)
            st["kv_len"][0] = c["Lk"]   # a batch is padded to its longest
            if c["Lq"] == c["Lk"]:
                st["q_len"] = st["kv_len"].clone()
        return st
    if c["op"] == "layernorm":
        t, s = _DT[c["dtype"]], (c["rows"], c["C"])
        return dict(case=c, x=(2.0 * randn(*s) + 0.5 * randn(1, c["C"])).to(t), dy=randn(*s).to(t), dres=randn(*s).to(t) if c["res"] else None,
                    gamma=1.0 + 0.2 * randn(c["C"]), beta=0.2 * randn(c["C"]))
    B, L, V, W = c["B"], c["L"], c["V"], c["W"]
    tok = (torch.rand(B, L, device="cuda", generator=g) ** 3 * V).long().clamp_(max=V - 1)   # a few words are frequent
    if c["pad"]:   # rows end in token 0
        n = (torch.rand(B, 1, device="cuda", generator=g) * 2 * (1 - c["pad"]) * L).long().clamp_(min=1)
        tok = torch.where(torch.arange(L, device="cuda")[None] < n, tok, 0)
    return dict(case=c, tokens=tok, table=randn(V, W).to(_DT[c["table"]]), pos=0.1 * randn(L, W) if c["pos"] else None,
                dy=randn(B, L, W).to(_DT[c["dtype"]]))


# ------------------------------------------------------------------------------------------------ plain forms
def _visible(c, st):
    """Which keys each query sees: bool [B, 1, Lq, Lk], or None for all."""
    Lq, Lk = c["Lq"], c["Lk"]
    if not c["causal"] and not c["ragged"]:
        return None
    i, j = torch.arange(Lq, device="cuda")[:, None], torch.arange(Lk, device="cuda")[None]
    m = (j <= i + Lk - Lq) if c["causal"] else (j >= 0) & (i >= 0)
    m = m[None, None]
    if st["kv_len"] is not None:
        m = m & (j < st["kv_len"][:, None, None, None])
    if st["q_len"] is not None:
        m = m & (i < st["q_len"][:, None, None, None])
    return m


def _attention(st):
    c, scale = st["case"], D ** -0.5
    rep = c["H"] // c["Hkv"]
    q, k, v = (st[n].float().transpose(1, 2) for n in ("q", "k", "v"))
    k, v = (t.repeat_interleave(rep, dim=1) for t in (k, v))
    s = torch.matmul(q, k.transpose(2, 3)) * scale
    vis = _visible(c, st)
    if vis is not None:
        s = s.masked_fill(~vis, float("-inf"))
    m = s.amax(dim=3, keepdim=True)
    m = torch.where(m == float("-inf"), 0.0, m)
    p = torch.exp(s - m)
    l = p.sum(dim=3, keepdim=True)
    lse = m + torch.log(l)
    p = p / torch.where(l == 0, 1.0, l)
    o = torch.matmul(p, v)
    t = st["q"].dtype
    out = dict(out=o.transpose(1, 2).to(t), lse=lse[..., 0])
    if c["dir"] == "fwd":
        return out
    do = st["dout"].float().transpose(1, 2)
    if st["q_len"] is not None:
        do = do * (torch.arange(c["Lq"], device="cuda")[:, None] < st["q_len"][:, None, None, None])
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = p * (torch.matmul(do, v.transpose(2, 3)) - (do * o).sum(dim=3, keepdim=True))
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3), q) * scale
    dk, dv = (t2.unflatten(1, (c["Hkv"], rep)).sum(dim=2) for t2 in (dk, dv))
    out.update(dq=dq.transpose(1, 2).to(t), dk=dk.transpose(1, 2).to(t), dv=dv.transpose(1, 2).to(t))
    return out


def _layernorm(st):
    c, t, x = st["case"], st["x"].dtype, st["x"].float()
    mean = x.mean(dim=1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).mean(dim=1, keepdim=True) + 1e-5)
    xh = xc * rstd
    out = dict(y=(xh * st["gamma"] + st["beta"]).to(t))
    if c["dir"] == "fwd":
        return out
    dy = st["dy"].float()
    a = dy * st["gamma"]
    dx = rstd * (a - a.mean(dim=1, keepdim=True) - xh * (a * xh).mean(dim=1, keepdim=True))
    if st["dres"] is not None:
        dx = dx + st["dres"].float()
    out.update(dx=dx.to(t), dgamma=(dy * xh).sum(dim=0), dbeta=dy.sum(dim=0))
    return out


def _embedding(st):
    c = st["case"]
    scale = c["W"] ** 0.5
    x = st["table"][st["tokens"]].float() * scale
    if st["pos"] is not None:
        x = x + st["pos"]
    out = dict(x=x.to(_DT[c["dtype"]]))
    if c["dir"] == "fwd":
        return out
    dy = st["dy"].float()
    out["dtable"] = torch.zeros(c["V"], c["W"], device="cuda").index_add_(0, st["tokens"].flatten(), dy.flatten(0, 1) * scale)
    if st["pos"] is not None:
        out["dpos"] = dy.sum(dim=0)
    return out


def run(st):
    c = st["case"]
    if not own:
        return {"attention": _attention, "layernorm": _layernorm, "embedding": _embedding}[c["op"]](st)
    from diffbir_amd import ops
    if c["op"] == "attention":
        lens = dict(causal=c["causal"], q_len=st["q_len"], kv_len=st["kv_len"])
        o, lse = ops.attention_fwd(st["q"], st["k"], st["v"], D ** -0.5, **lens)
        out = dict(out=o, lse=lse)
        if c["dir"] == "step":
            out["dq"], out["dk"], out["dv"] = ops.attention_bwd(st["dout"], st["q"], st["k"], st["v"], o, lse, D ** -0.5, **lens)
        return out
    if c["op"] == "layernorm":
        y, stats = ops.layernorm_fwd(st["x"], st["gamma"], st["beta"], eps=1e-5)
        out = dict(y=y)
        if c["dir"] == "step":
            out["dx"], out["dgamma"], out["dbeta"] = ops.layernorm_bwd(st["dy"], st["x"], st["gamma"], stats, dres=st["dres"])
        return out
    scale = c["W"] ** 0.5
    out = dict(x=ops.embedding(st["tokens"], st["table"], scale=scale, pos=st["pos"], dtype=_DT[c["dtype"]]))
    if c["dir"] == "step":
        out["dtable"], dpos = ops.embedding_bwd(st["dy"], st["tokens"], c["V"], scale=scale, pos_rows=c["L"] if c["pos"] else 0)
        if dpos is not None:
            out["dpos"] = dpos
    return out


def work(case):
    c, size = case, {"f16": 2, "bf16": 2, "f32": 4}[case["dtype"]]
    step = c["dir"] == "step"
    if c["op"] == "attention":
        Lq, Lk = c["Lq"], c["Lk"]
        pairs = float(sum(max(0, min(Lk, i + 1 + Lk - Lq)) for i in range(Lq))) if c["causal"] else float(Lq) * Lk
        if c["ragged"]:   # lengths are uniform: 1/2 of the keys, 1/3 of the pairs where queries are cut alike
            pairs *= (1 / 3 if Lq == Lk else 1 / 2)
        nq, nk = c["B"] * c["H"] * Lq * D, c["B"] * c["Hkv"] * Lk * D
        return dict(bytes=size * (nq * (4 if step else 2) + nk * (4 if step else 2)) + 4 * nq // D,
                    flops=c["B"] * c["H"] * pairs * D * (14 if step else 4))
    if c["op"] == "layernorm":
        n = c["rows"] * c["C"]
        return dict(bytes=size * n * (2 + step * (2 + c["res"])) + 8 * c["C"] * (1 + step), flops=n * (8 + 12 * step))
    n, tw = c["B"] * c["L"], {"f16": 2, "bf16": 2, "f32": 4}[c["table"]]
    rows = min(c["V"], n * (1 - c["pad"]) + 1)   # about as many rows of the table are read
    return dict(bytes=rows * c["W"] * tw + n * (8 + c["W"] * size * (1 + step)) + c["pos"] * c["L"] * c["W"] * 4 * (1 + step)
                + step * 4 * c["V"] * c["W"], flops=n * c["W"] * (2 + 2 * step))


def exact(case, seed):
    """In 64 bits from the definitions, one sample and head (or a block of rows) at a time."""
    c, st = case, prepare(case, seed)
    if c["op"] == "attention":
        B, H, Hkv, Lq, Lk = (c[n] for n in ("B", "H", "Hkv", "Lq", "Lk"))
        q, k, v, do = (st[n].double() for n in ("q", "k", "v", "dout"))
        out = dict(out=torch.zeros_like(q), lse=torch.full((B, H, Lq), float("-inf"), device="cuda", dtype=torch.float64))
        if c["dir"] == "step":
            out.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
        nk = [Lk] * B if st["kv_len"] is None else st["kv_len"].tolist()
        nq = [Lq] * B if st["q_len"] is None else st["q_len"].tolist()
        for b in range(B):
            first = max(0, Lq - Lk) if c["causal"] else 0   # queries above see no key
            if nk[b] == 0 or nq[b] <= first:
                continue
            for h in range(H):
                g = h // (H // Hkv)
                Q, K, V = q[b, first:nq[b], h], k[b, :nk[b], g].contiguous(), v[b, :nk[b], g].contiguous()
                z = (Q @ K.T) / D ** 0.5
                if c["causal"]:
                    last = torch.arange(first, nq[b], device="cuda") + Lk - Lq
                    z[torch.arange(nk[b], device="cuda")[None] > last[:, None]] = float("-inf")
                lse = torch.logsumexp(z, dim=1)
                P = torch.exp(z - lse[:, None])
                O = P @ V
                out["out"][b, first:nq[b], h], out["lse"][b, h, first:nq[b]] = O, lse
                if c["dir"] == "step":
                    G = do[b, first:nq[b], h]
                    Z = P * (G @ V.T - (G * O).sum(1, keepdim=True)) / D ** 0.5
                    out["dq"][b, first:nq[b], h] = Z @ K
                    out["dk"][b, :nk[b], g] += Z.T @ Q
                    out["dv"][b, :nk[b], g] += P.T @ G
        return out
    if c["op"] == "layernorm":
        x = st["x"].double()
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        std = (var + 1e-5).sqrt()
        xh = (x - mean) / std
        out = dict(y=xh * st["gamma"].double() + st["beta"].double())
        if c["dir"] == "step":
            dy = st["dy"].double()
            out["dgamma"], out["dbeta"] = (dy * xh).sum(0), dy.sum(0)
            a = dy * st["gamma"].double()
            dx = (a - (a.sum(1, keepdim=True) + xh * (a * xh).sum(1, keepdim=True)) / c["C"]) / std
            out["dx"] = dx if st["dres"] is None else dx + st["dres"].double()
        return out
    scale, W = c["W"] ** 0.5, c["W"]
    rows = st["table"].double().index_select(0, st["tokens"].flatten()).reshape(c["B"], c["L"], W) * scale
    out = dict(x=rows if st["pos"] is None else rows + st["pos"].double())
    if c["dir"] == "step":
        dy = st["dy"].double()
        order = st["tokens"].flatten().argsort(stable=True)
        ids, n = st["tokens"].flatten()[order].unique_consecutive(return_counts=True)
        ends = dy.reshape(-1, W)[order].cumsum(0)[n.cumsum(0) - 1]
        out["dtable"] = torch.zeros(c["V"], W, device="cuda", dtype=torch.float64)
        out["dtable"][ids] = torch.diff(ends, dim=0, prepend=torch.zeros_like(ends[:1])) * scale
        if st["pos"] is not None:
            out["dpos"] = dy.sum(0)
    return out
