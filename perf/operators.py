"""Cases and plain forms of the encoder and softmax-loss operators (`ops.linear_act`, `ops.packed_attention`,
`ops.softmax_loss` and their backward passes).

`run` computes a case either in its plain form — elementary torch operations in 32 bits — or, with `own` set, through the
framework's entry points; `exact` evaluates the operator's definition in 64 bits.

Formulas (T tokens, documents packed back to back; all sums over the last axis unless named):

    linear_act        z = x W^T + b,  y = act(z) + r
                      dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum_rows dz   (dr = dy: the caller has it)
    packed_attention  s_ij = cap tanh(scale q_i.k_j / cap) - slope_h |i - j|   over the keys j that query i may see: those of
                      its own document, not taken out by the key mask, and with "causal" j <= i, with "prefix" j <= i or
                      j < prefix(document);  o_i = sum_j softmax_j(s_ij) v_j, 0 for a query that sees no key
    softmax_loss      l_ij = scale x_i.w_j over the candidates j that share no group id with row i, and its target;
                      loss_i = log sum_j exp l_ij - l_i,target  (0 for a row whose target is IGNORE);
                      with upstream c_i per row: dx = scale G w, dw = scale G^T x,  G_ij = c_i (p_ij - [j = target_i])
"""
import math
import random

import torch

own = False

IGNORE = -100
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
WIDTH = {"f32": 4, "bf16": 2, "f16": 2}


# --------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one query of a few tokens through the feed-forward's first product: what a search request waits for
        dict(name="linear_one_query", op="linear", dtype="f32", train=False, M=11, K=384, N=1536, act="gelu", bias=True, res=False),
        # 512 passages of ~70 tokens through the frozen encoder in fp32, the framework's parity type
        dict(name="linear_passages_f32", op="linear", dtype="f32", train=False, M=35841, K=384, N=1536, act="gelu", bias=True, res=False),
        # the feed-forward's second product with its residual, 16 bits: the encoder_autocast="bf16" pass over a corpus chunk
        dict(name="linear_down_bf16", op="linear", dtype="bf16", train=False, M=35841, K=1536, N=384, act="none", bias=True, res=True),
        # a training step's product and its three gradients at a wider encoder
        dict(name="linear_train_bf16", op="linear", dtype="bf16", train=True, M=16384, K=1024, N=4096, act="gelu", bias=True, res=True),
        # one query's attention: eleven tokens, twelve heads
        dict(name="attention_one_query", op="attention", dtype="f32", train=False, docs=1, lo=11, hi=11, H=12, Hkv=12, Dh=32,
             mask="full", cap=0.0, alibi=False, holes=False),
        # 512 passages as the feature cache encodes them, fp32
        dict(name="attention_passages_f32", op="attention", dtype="f32", train=False, docs=512, lo=12, hi=128, H=12, Hkv=12, Dh=32,
             mask="full", cap=0.0, alibi=False, holes=False),
        # a few long documents, prefix visible to all, capped scores, a distance bias and masked keys together
        dict(name="attention_long_bf16", op="attention", dtype="bf16", train=False, docs=5, lo=1001, hi=4096, H=12, Hkv=12, Dh=64,
             mask="prefix", cap=30.0, alibi=True, holes=True),
        # a training batch of mixed lengths, both directions, 16 bits
        dict(name="attention_train_bf16", op="attention", dtype="bf16", train=True, docs=256, lo=8, hi=512, H=12, Hkv=12, Dh=32,
             mask="full", cap=0.0, alibi=True, holes=False),
        # causal documents with heads shared four to one, fp16, both directions
        dict(name="attention_train_f16", op="attention", dtype="f16", train=True, docs=16, lo=700, hi=2048, H=16, Hkv=4, Dh=128,
             mask="causal", cap=0.0, alibi=False, holes=False),
        # every other document of the batch is a candidate: the in-batch softmax loss on unit rows, temperature 1/20
        dict(name="softmax_inbatch_f32", op="softmax", dtype="f32", train=True, N=2048, V=2048, D=384, scale=20.0, unit=True, groups=True),
        # a large vocabulary of candidates, both directions, 16 bits
        dict(name="softmax_vocab_bf16", op="softmax", dtype="bf16", train=True, N=8192, V=30522, D=384, scale=1.0, unit=False, groups=False),
        # validation: loss only, few queries over every passage of a corpus
        dict(name="softmax_corpus_bf16", op="softmax", dtype="bf16", train=False, N=203, V=250000, D=384, scale=20.0, unit=True, groups=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        dtype = rng.choice(["f32", "bf16", "f16"])
        op = rng.choice(["linear", "attention", "softmax"])
        train = rng.random() < 0.5
        if op == "linear":
            K, N = _log(rng, 64, 2048), _log(rng, 64, 4096)
            if rng.random() < 0.7:  # widths are multiples of 8 more often than not
                K, N = max(64, K // 8 * 8), max(64, N // 8 * 8)
            case = dict(op=op, dtype=dtype, train=train, M=_log(rng, 1, 40000), K=K, N=N,
                        act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.8, res=rng.random() < 0.5)
            ok = case["M"] * K * N <= 16384 * 1024 * 4096 // (4 if dtype == "f32" else 1)
        elif op == "attention":
            hi = _log(rng, 1, 4096)
            H = rng.choice([4, 8, 12, 16])
            case = dict(op=op, dtype=dtype, train=train, docs=_log(rng, 1, 512), lo=max(1, int(hi * rng.random())), hi=hi, H=H,
                        Hkv=rng.choice([H, H, H // 2, H // 4]), Dh=rng.choice([32, 64, 128]), mask=rng.choice(["full", "full", "causal", "prefix"]),
                        cap=rng.choice([0.0, 0.0, 30.0]), alibi=rng.random() < 0.4, holes=rng.random() < 0.4)
            ok = case["docs"] * hi * hi * H <= (16 * 2048 * 2048 * 16 if not train else 16 * 2048 * 2048 * 8) and \
                case["docs"] * hi * H * case["Dh"] <= 1 << 28
        else:
            case = dict(op=op, dtype=dtype, train=train, N=_log(rng, 1, 8192), V=_log(rng, 2, 250000), D=_log(rng, 64, 768) // 8 * 8,
                        scale=20.0, unit=True, groups=rng.random() < 0.4)
            if rng.random() < 0.5:
                case.update(scale=1.0, unit=False)
            ok = case["N"] * case["V"] * case["D"] <= 8192 * 30522 * 384 // (4 if dtype == "f32" else 1)
        if ok:
            return case


# --------------------------------------------------------------------------------------------------- inputs
def _layout(case):
    """Document lengths and prefixes of an attention case: a function of the case alone (its work depends on them)."""
    r = random.Random(case["docs"] * 1000003 + case["lo"] * 1009 + case["hi"])
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["docs"])]
    lens[0] = case["hi"]
    prefix = [r.randint(0, max(1, n // 2)) for n in lens]
    return lens, prefix


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dt)

    st = dict(case=case)
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        # normalised activations, weights of the usual 1/sqrt(K) size
        st["x"], st["w"] = randn(M, K), randn(N, K, std=K ** -0.5)
        st["b"] = randn(N, std=0.1) if case["bias"] else None
        st["r"] = randn(M, N) if case["res"] else None
        st["dy"] = randn(M, N) if case["train"] else None
    elif case["op"] == "attention":
        lens, prefix = _layout(case)
        H, Hkv, Dh = case["H"], case["Hkv"], case["Dh"]
        T = sum(lens)
        qkv = randn(T, H + 2 * Hkv, Dh)  # one fused projection's output: q, k, v are its column blocks
        st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
        cu = torch.tensor([0] + lens).cumsum(0)
        st["cu"] = cu.to(torch.int32).cuda()
        st["prefix"] = torch.tensor(prefix, dtype=torch.int32).cuda() if case["mask"] == "prefix" else None
        st["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda") if case["alibi"] else None
        st["keep"] = (torch.rand(T, generator=g, device="cuda") > 0.1) if case["holes"] else None
        st["do"] = randn(T, H, Dh) if case["train"] else None
        st["lens"] = lens
        # padded rows of the plain form: token t sits at (document, position)
        L = max(lens)
        doc = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
        st["slot"] = (doc * L + torch.arange(T) - cu[:-1][doc]).cuda()
    else:
        N, V, D = case["N"], case["V"], case["D"]
        x = torch.randn(N, D, generator=g, device="cuda")
        w = torch.randn(V, D, generator=g, device="cuda")
        st["t"] = torch.randint(0, V, (N,), generator=g, device="cuda")
        if case["unit"]:  # cosine similarities: a query lies near its document
            if N == V:
                st["t"] = torch.arange(N, device="cuda")
            x = x + 0.7 * w[st["t"]]
            x, w = x / x.norm(dim=1, keepdim=True), w / w.norm(dim=1, keepdim=True)
        else:
            w *= 2.0 * D ** -0.5
        st["x"], st["w"] = x.to(dt), w.to(dt)
        st["rid"] = st["cid"] = None
        if case["groups"]:  # about two documents of each query id
            st["cid"] = torch.randint(0, max(1, V // 2), (V,), generator=g, device="cuda")
            st["rid"] = st["cid"][st["t"]]
        if N > 4 and not case["unit"]:
            st["t"][::17] = IGNORE  # positions that carry no label
        # the mean's upstream gradient, behind a loss scaler where the type needs one
        st["c"] = torch.full((N,), (65536.0 if case["dtype"] == "f16" else 1.0) / N, device="cuda") if case["train"] else None
    torch.cuda.synchronize()
    return st


# --------------------------------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "attention": _own_attention, "softmax": _own_softmax}[op](state)
    return {"linear": _plain_linear, "attention": _plain_attention, "softmax": _plain_softmax}[op](state)


def _own_linear(st):
    from two_towers_overlords_amd import ops

    act = st["case"]["act"]
    if not st["case"]["train"]:
        return ops.linear_act(st["x"], st["w"], st["b"], st["r"], act)
    y, z = ops.linear_act(st["x"], st["w"], st["b"], st["r"], act, save_preact=True)
    dx, dw, db = ops.linear_act_bwd(st["dy"], st["x"], st["w"], z, act, bias=st["b"] is not None)
    return [y, dx, dw] + ([db] if st["b"] is not None else [])


def _own_attention(st):
    from two_towers_overlords_amd import ops

    c = st["case"]
    kw = dict(causal=c["mask"] == "causal", prefix=st["prefix"], softcap=c["cap"], slopes=st["slopes"], key_mask=st["keep"])
    o, lse = ops.packed_attention(st["q"], st["k"], st["v"], st["cu"], **kw)
    if not c["train"]:
        return o
    return [o, *ops.packed_attention_bwd(st["do"], st["q"], st["k"], st["v"], o, lse, st["cu"], **kw)]


def _own_softmax(st):
    from two_towers_overlords_amd import ops

    kw = dict(scale=st["case"]["scale"], row_ids=st["rid"], cand_ids=st["cid"], ignore_index=IGNORE)
    loss, lse = ops.softmax_loss(st["x"], st["w"], st["t"], **kw)
    if not st["case"]["train"]:
        return [loss, lse]
    return [loss, *ops.softmax_loss_bwd(st["c"], st["x"], st["w"], st["t"], lse, **kw)]


# --------------------------------------------------------------------------------------------------- plain forms
def _act(z, act):
    """(act(z), act'(z))"""
    if act == "none":
        return z, None
    if act == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    if act == "gelu":
        phi = 0.5 * (1.0 + torch.erf(z * 0.7071067811865476))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    if act == "gelu_tanh":
        t = torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * 0.7978845608028654 * (1.0 + 0.134145 * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return z * s, s * (1.0 + z * (1.0 - s))


def _plain_linear(st):
    dt = st["x"].dtype
    x, w = st["x"].float(), st["w"].float()
    z = x @ w.t()
    if st["b"] is not None:
        z = z + st["b"].float()
    y, dact = _act(z, st["case"]["act"])
    if st["r"] is not None:
        y = y + st["r"].float()
    y = y.to(dt)
    if not st["case"]["train"]:
        return y
    dz = st["dy"].float()
    if dact is not None:
        dz = dz * dact
    out = [y, (dz @ w).to(dt), (dz.t() @ x).to(dt)]
    if st["b"] is not None:
        out.append(dz.sum(0).to(dt))
    return out


def _plain_attention(st):
    c, dt = st["case"], st["q"].dtype
    H, Hkv, Dh = c["H"], c["Hkv"], c["Dh"]
    n, L, slot = len(st["lens"]), max(st["lens"]), st["slot"]
    dev = slot.device

    def pad(t, rep):  # [T, h, Dh] -> [n * H, L, Dh]
        p = torch.zeros(n * L, t.shape[1], Dh, device=dev)
        p[slot] = t.float()
        p = p.view(n, L, t.shape[1], Dh).transpose(1, 2)
        if rep > 1:
            p = p.unsqueeze(2).expand(n, t.shape[1], rep, L, Dh)
        return p.reshape(n * H, L, Dh).contiguous()

    def unpad(p):  # [n * H, L, Dh] -> [T, H, Dh]
        return p.view(n, H, L, Dh).transpose(1, 2).reshape(n * L, H, Dh)[slot]

    rep = H // Hkv
    q, k, v = pad(st["q"], 1), pad(st["k"], rep), pad(st["v"], rep)
    i = torch.arange(L, device=dev)
    live = torch.zeros(n * L, dtype=torch.bool, device=dev)
    live[slot] = True if st["keep"] is None else st["keep"]
    see = live.view(n, 1, L).expand(n, L, L)
    if c["mask"] == "causal":
        see = see & (i[None, :] <= i[:, None])
    elif c["mask"] == "prefix":
        see = see & ((i[None, :] <= i[:, None])[None] | (i[None, None, :] < st["prefix"].view(n, 1, 1)))
    see = see.unsqueeze(1)
    scale = Dh ** -0.5
    s = torch.bmm(q, k.transpose(1, 2).contiguous()) * scale
    th = None
    if c["cap"] > 0:
        th = torch.tanh(s / c["cap"])
        s = c["cap"] * th
    s = s.view(n, H, L, L)
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, H, 1, 1) * (i[None, :] - i[:, None]).abs()
    s = torch.where(see, s, torch.full((), -math.inf, device=dev))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(s - m)
    del s
    den = p.sum(-1, keepdim=True)
    p = (p / torch.where(den == 0, torch.ones_like(den), den)).view(n * H, L, L)
    o = torch.bmm(p, v)
    out = unpad(o).to(dt)
    if not c["train"]:
        return out
    do = pad(st["do"], 1)
    dv = torch.bmm(p.transpose(1, 2).contiguous(), do)
    dp = torch.bmm(do, v.transpose(1, 2).contiguous())
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    if th is not None:
        ds = ds * (1.0 - th * th)
    dq = torch.bmm(ds, k)
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), q)

    def group(t):  # sum over the query heads that share a key head
        return unpad(t).view(-1, Hkv, rep, Dh).sum(2).to(dt)

    return [out, unpad(dq).to(dt), group(dk), group(dv)]


def _plain_softmax(st):
    c, dt = st["case"], st["x"].dtype
    x, w, t = st["x"].float(), st["w"].float(), st["t"]
    on = t != IGNORE
    tt = torch.where(on, t, torch.zeros_like(t)).unsqueeze(1)
    l = (x @ w.t()) * c["scale"]
    if st["rid"] is not None:
        out = st["rid"].unsqueeze(1) == st["cid"].unsqueeze(0)
        out.scatter_(1, tt, False)
        l = torch.where(out, torch.full((), -math.inf, device=l.device), l)
    m = l.amax(1, keepdim=True)
    lt = l.gather(1, tt)
    p = torch.exp(l - m)
    del l
    den = p.sum(1, keepdim=True)
    lse = torch.log(den) + m
    loss = torch.where(on, (lse - lt).squeeze(1), torch.zeros((), device=x.device))
    if not c["train"]:
        return [loss, lse.squeeze(1)]
    p = p / den
    p.scatter_add_(1, tt, torch.full_like(lt, -1.0))
    p = p * (st["c"] * on * c["scale"]).unsqueeze(1)
    return [loss, (p @ w).to(dt), (p.t() @ x).to(dt)]


# --------------------------------------------------------------------------------------------------- work
def work(case):
    b = WIDTH[case["dtype"]]
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        n = M * K + N * K + M * N + (N if case["bias"] else 0) + (M * N if case["res"] else 0)
        if case["train"]:
            n += M * N + M * K + N * K + (N if case["bias"] else 0)
        return {"bytes": n * b, "flops": (6 if case["train"] else 2) * M * K * N}
    if case["op"] == "attention":
        lens, prefix = _layout(case)
        H, Hkv, Dh = case["H"], case["Hkv"], case["Dh"]
        pairs = 0
        for n, p in zip(lens, prefix):
            if case["mask"] == "full":
                pairs += n * n
            else:  # query i sees max(i + 1, p) keys
                p = min(p, n) if case["mask"] == "prefix" else 0
                pairs += p * p + (n * (n + 1) - p * (p + 1)) // 2
        T = sum(lens)
        n = T * (2 * H + 2 * Hkv) * Dh
        if case["train"]:
            n += T * (2 * H + 2 * Hkv) * Dh
        return {"bytes": n * b, "flops": (14 if case["train"] else 4) * pairs * H * Dh}
    N, V, D = case["N"], case["V"], case["D"]
    n = (N + V) * D * b * (2 if case["train"] else 1) + N * 12 + (8 * (N + V) if case["groups"] else 0)
    return {"bytes": n, "flops": (6 if case["train"] else 2) * N * V * D}


# --------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.enable_grad():
        return {"linear": _exact_linear, "attention": _exact_attention, "softmax": _exact_softmax}[case["op"]](st)


def _leaf(t):
    return None if t is None else t.detach().double().requires_grad_(True)


def _exact_linear(st):
    c = st["case"]
    x, w, b, r = _leaf(st["x"]), _leaf(st["w"]), _leaf(st["b"]), _leaf(st["r"])
    z = torch.mm(x, w.transpose(0, 1))
    z = z if b is None else z + b
    if c["act"] == "relu":
        y = z.clamp(min=0)
    elif c["act"] == "gelu":
        y = z * torch.erfc(-z / math.sqrt(2.0)) / 2
    elif c["act"] == "gelu_tanh":
        y = z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    elif c["act"] == "silu":
        y = z / (1 + torch.exp(-z))
    else:
        y = z
    y = y if r is None else y + r
    if not c["train"]:
        return y.detach()
    leaves = [t for t in (x, w, b) if t is not None]
    return [y.detach(), *torch.autograd.grad(y, leaves, st["dy"].double())]


def _exact_attention(st):
    c = st["case"]
    H, Hkv, Dh = c["H"], c["Hkv"], c["Dh"]
    outs, grads, at = [], [], 0
    for d, n in enumerate(st["lens"]):
        rows = slice(at, at + n)
        at += n
        q, k, v = (_leaf(st[name][rows]) for name in ("q", "k", "v"))
        pos = torch.arange(n, device=q.device, dtype=torch.float64)
        hidden = torch.zeros(n, n, dtype=torch.bool, device=q.device)
        if c["mask"] != "full":
            hidden |= pos.view(1, n) > pos.view(n, 1)
        if c["mask"] == "prefix":
            hidden &= pos.view(1, n) >= st["prefix"][d].double()
        if st["keep"] is not None:
            hidden |= ~st["keep"][rows].view(1, n)
        out = []
        for h in range(H):
            kv = h // (H // Hkv)
            s = torch.mm(q[:, h], k[:, kv].t()) / math.sqrt(Dh)
            if c["cap"] > 0:
                s = torch.tanh(s / c["cap"]) * c["cap"]
            if st["slopes"] is not None:
                s = s - (pos.view(n, 1) - pos.view(1, n)).abs() * st["slopes"][h].double()
            s = s.masked_fill(hidden, -1e300)  # rows that see nothing are zeroed below
            p = torch.softmax(s, 1).masked_fill(hidden, 0.0)
            out.append(torch.mm(p, v[:, kv]))
        o = torch.stack(out, 1)
        outs.append(o.detach())
        if c["train"]:
            grads.append(torch.autograd.grad(o, (q, k, v), st["do"][rows].double()))
        if c["docs"] * H > 1000 and d > 0 and d % 64 == 0:
            torch.cuda.empty_cache()
    if not c["train"]:
        return torch.cat(outs)
    return [torch.cat(outs)] + [torch.cat([g[i] for g in grads]) for i in range(3)]


def _exact_softmax(st):
    c = st["case"]
    x, w, t = _leaf(st["x"]), _leaf(st["w"]), st["t"]
    N, V = x.shape[0], w.shape[0]
    step = max(1, min(N, (1 << 27) // V))  # rows at a time: about 1 GB of logits
    losses, lses, dx, dw = [], [], [], torch.zeros_like(w) if c["train"] else None
    for a in range(0, N, step):
        xr, tr = x[a:a + step].detach().requires_grad_(c["train"]), t[a:a + step]
        on = tr != IGNORE
        at = torch.where(on, tr, torch.zeros_like(tr))
        l = torch.mm(xr, w.t()) * c["scale"]
        if st["rid"] is not None:
            same = st["rid"][a:a + step].view(-1, 1) == st["cid"].view(1, -1)
            same &= torch.arange(V, device=w.device).view(1, -1) != at.view(-1, 1)
            l = l.masked_fill(same, -math.inf)
        lse = torch.logsumexp(l, 1)
        loss = (lse - l[torch.arange(len(at), device=w.device), at]).masked_fill(~on, 0.0)
        losses.append(loss.detach())
        lses.append(lse.detach())
        if c["train"]:
            gx, gw = torch.autograd.grad(loss, (xr, w), st["c"][a:a + step].double())
            dx.append(gx)
            dw += gw
    if not c["train"]:
        return [torch.cat(losses), torch.cat(lses)]
    return [torch.cat(losses), torch.cat(dx), dw]
