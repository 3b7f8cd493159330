"""The operators of a served attention layer: cases, plain forms and the framework's calls.

  lora          a shared projection with the low-rank adapters of many requests beside it
  qk_norm_rope  norms of queries and keys for each head and the position rotation, in one pass
  attn_prompt   attention over packed prompts with grouped heads, single tokens included

`run` computes an operator in elementary torch operations where `own` is false, and through
`hopper_gemm_b200`'s public functions where it is true.
"""
import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-6


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # One user's next token through an output projection: one request, one adapter.
        dict(name="lora_token", op="lora", T=1, K=4096, N=4096, rank=16, segs=1, adapters=1,
             plain=0, cut=1),
        # A decoding batch: 48 requests with one token each over 32 adapters of the fused
        # query/key/value projection, every eighth request without an adapter.
        dict(name="lora_decode48", op="lora", T=48, K=4096, N=6144, rank=32, segs=48,
             adapters=32, plain=8, cut=2),
        # Prompts being filled in while others decode: 40 requests of uneven lengths, odd total.
        dict(name="lora_mixed1037", op="lora", T=1037, K=4096, N=4096, rank=64, segs=40,
             adapters=12, plain=6, cut=3),
        # Long prompts of six requests through the fused query/key/value projection.
        dict(name="lora_prompt8192", op="lora", T=8192, K=4096, N=6144, rank=64, segs=6,
             adapters=4, plain=0, cut=4),
        # The decoding batch's queries and keys after the projection.
        dict(name="norm_decode48", op="norm", T=48, heads_q=32, heads_kv=8, dim=128, rot=128,
             axes=1, interleaved=False, far=32768, cut=1),
        # A packed prompt of odd length.
        dict(name="norm_prompt8191", op="norm", T=8191, heads_q=32, heads_kv=8, dim=128, rot=128,
             axes=1, interleaved=False, far=8192, cut=2),
        # Image and video tokens: positions in time, height and width, a part of each head turned.
        dict(name="norm_video2500", op="norm", T=2500, heads_q=16, heads_kv=16, dim=80, rot=64,
             axes=3, interleaved=True, far=4096, cut=3),
        # Sixteen short questions, packed: launch and tail latency count.
        dict(name="attn_short16", op="attn", batch=16, q_total=1021, past=0, heads_q=32,
             heads_kv=8, dim=128, causal=True, cut=1),
        # A dozen prompts of uneven lengths in one packed batch.
        dict(name="attn_ragged12", op="attn", batch=12, q_total=8192, past=0, heads_q=32,
             heads_kv=8, dim=128, causal=True, cut=2),
        # One long prompt.
        dict(name="attn_long16384", op="attn", batch=1, q_total=16384, past=0, heads_q=32,
             heads_kv=8, dim=128, causal=True, cut=3),
        # One new token for each of 16 requests over keys of up to about 16000 tokens.
        dict(name="attn_token16", op="attn", batch=16, q_total=16, past=131072, heads_q=32,
             heads_kv=8, dim=128, causal=True, cut=4),
        # Prompts appended to earlier turns: fewer, smaller heads, no group.
        dict(name="attn_append5", op="attn", batch=5, q_total=3001, past=9000, heads_q=16,
             heads_kv=16, dim=64, causal=True, cut=5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["lora", "norm", "attn", "lora", "attn"])
    cut = rng.randrange(1, 1 << 20)
    if op == "lora":
        T = _log_int(rng, 1, 8192)
        K, N = 8 * _log_int(rng, 64, 1024), 8 * _log_int(rng, 64, 1024)
        while T * K * N > 8192 * 4096 * 6144:
            T = (T + 1) // 2
        return dict(op=op, T=T, K=K, N=N, rank=rng.choice([8, 16, 24, 32, 64, 128]),
                    segs=_log_int(rng, 1, min(T, 96)), adapters=_log_int(rng, 1, 48),
                    plain=rng.choice([0, 0, 3, 5]), cut=cut)
    if op == "norm":
        heads_kv = rng.choice([1, 2, 4, 8, 16])
        dim = rng.choice([64, 80, 96, 128, 256])
        T = _log_int(rng, 1, 16384 * 128 // dim)
        group = rng.choice([1, 2, 3, 4, 7])
        while T * heads_kv * (group + 1) * dim > 8191 * 40 * 128:
            T = (T + 1) // 2
        rot = rng.choice([dim, dim, dim // 2]) // 16 * 16
        return dict(op=op, T=T, heads_q=heads_kv * group, heads_kv=heads_kv, dim=dim, rot=rot,
                    axes=rng.choice([1, 1, 2, 3]), interleaved=rng.random() < 0.4,
                    far=_log_int(rng, 16, 1 << 20), cut=cut)
    heads_kv = rng.choice([1, 2, 4, 8])
    heads_q = heads_kv * rng.choice([1, 2, 3, 4, 7, 8])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128])
    batch = _log_int(rng, 1, 48)
    if rng.random() < 0.3:
        q_total, past = batch, _log_int(rng, 64, 131072)
    else:
        q_total = _log_int(rng, batch, 12288)
        past = rng.choice([0, 0, _log_int(rng, 16, 8192)])
    case = dict(op=op, batch=batch, q_total=q_total, past=past, heads_q=heads_q,
                heads_kv=heads_kv, dim=dim, causal=rng.random() < 0.8, cut=cut)
    top = 32 * 128 * 16384 * 16384 // 2
    while heads_q * dim * case["q_total"] * (case["q_total"] + case["past"]) > top:
        case["q_total"] = max(1, case["q_total"] // 2)
        case["past"] //= 2
    return case


def _cut(total, parts, cut):
    """`total` tokens in `parts` uneven lengths; an empty one among them where there are many."""
    rng = random.Random(cut)
    w = [rng.random() ** 2 + 0.02 for _ in range(parts)]
    if parts > 6 and total > parts:
        w[rng.randrange(parts)] = 0.0
    s = sum(w)
    lens = [int(total * x / s) for x in w]
    lens[max(range(parts), key=lambda i: w[i])] += total - sum(lens)
    return lens


def _lora_plan(case):
    T, segs = case["T"], case["segs"]
    lens = [1] * T if segs == T else _cut(T, segs, case["cut"])
    rng = random.Random(case["cut"] + 7)
    ids = [rng.randrange(case["adapters"]) for _ in lens]
    if case["plain"]:
        ids = [-1 if i % case["plain"] == case["plain"] - 1 else a for i, a in enumerate(ids)]
    return lens, ids


def _attn_plan(case):
    B, q_total = case["batch"], case["q_total"]
    q = [1] * B if q_total == B else _cut(q_total, B, case["cut"])
    past = _cut(case["past"], B, case["cut"] + 13) if case["past"] else [0] * B
    return q, [a + b for a, b in zip(q, past)]


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _pairs(case):
    """Query/key pairs of one head that the mask leaves."""
    n = 0
    for q, k in zip(*_attn_plan(case)):
        n += q * k - (q * (q - 1) // 2 if case["causal"] else 0)
    return n


def work(case):
    if case["op"] == "lora":
        T, K, N, r = case["T"], case["K"], case["N"], case["rank"]
        lens, ids = _lora_plan(case)
        used = len({a for n, a in zip(lens, ids) if n and a >= 0})
        rows = sum(n for n, a in zip(lens, ids) if a >= 0)
        return dict(bytes=2 * (T * K + K * N + T * N + used * r * (K + N)),
                    flops=2 * T * K * N + 2 * rows * r * (K + N))
    if case["op"] == "norm":
        n = case["T"] * (case["heads_q"] + case["heads_kv"]) * case["dim"]
        return dict(bytes=4 * n + 4 * case["T"] * case["axes"], flops=8 * n)
    q, k = _attn_plan(case)
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["dim"]
    return dict(bytes=2 * d * (2 * sum(q) * hq + 2 * sum(k) * hkv), flops=4 * d * hq * _pairs(case))


# ------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(shape, std=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * std).half()

    st = dict(case=case)
    if case["op"] == "lora":
        T, K, N, r, A = (case[x] for x in ("T", "K", "N", "rank", "adapters"))
        lens, ids = _lora_plan(case)
        st.update(X=normal((T, K)), W=normal((K, N), K ** -0.5), down=normal((A, K, r), K ** -0.5),
                  up=normal((A, r, N), 0.5 * r ** -0.5),
                  scale=torch.rand(A, generator=g, device=DEV) + 0.5, lens=lens, ids=ids,
                  seg_start=torch.tensor(_starts(lens), dtype=torch.int32, device=DEV),
                  seg_adapter=torch.tensor(ids, dtype=torch.int32, device=DEV))
    elif case["op"] == "norm":
        T, hq, hkv, d, rot = (case[x] for x in ("T", "heads_q", "heads_kv", "dim", "rot"))
        # Queries and keys are views into the rows of the fused projection.
        qkv = normal((T, hq + 2 * hkv, d), 1.5)
        pos = torch.randint(0, case["far"], (case["axes"], T), generator=g, device=DEV,
                            dtype=torch.int32)
        if case["axes"] == 1:
            pos = pos.sort(dim=1).values.contiguous()
        inv = torch.tensor([10000.0 ** (-2 * i / rot) for i in range(rot // 2)],
                           dtype=torch.float32, device=DEV)
        axis = [i * case["axes"] // (rot // 2) for i in range(rot // 2)]
        st.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], wq=normal((d,), 0.1) + 1,
                  wk=normal((d,), 0.1) + 1, pos=pos, inv=inv, axis_list=axis,
                  axis=torch.tensor(axis, dtype=torch.uint8, device=DEV))
    else:
        hq, hkv, d = case["heads_q"], case["heads_kv"], case["dim"]
        q, k = _attn_plan(case)
        # Values of a normed head: every score has a spread of about one after the scale.
        if case["past"]:
            st.update(q=normal((sum(q), hq, d)), k=normal((sum(k), hkv, d)),
                      v=normal((sum(k), hkv, d)))
        else:
            qkv = normal((sum(q), hq + 2 * hkv, d))
            st.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:])
        st.update(q_lens=q, k_lens=k,
                  cu_q=torch.tensor(_starts(q), dtype=torch.int32, device=DEV),
                  cu_k=torch.tensor(_starts(k), dtype=torch.int32, device=DEV))
    return st


# ------------------------------------------------------------------------------- plain forms
def _plain_lora(st):
    x = st["X"].float()
    y = x @ st["W"].float()
    at = 0
    for n, a in zip(st["lens"], st["ids"]):
        if n and a >= 0:
            h = x[at:at + n] @ st["down"][a].float()
            y[at:at + n] += st["scale"][a] * (h @ st["up"][a].float())
        at += n
    return y.half()


def _plain_turn(x, w, cos, sin, rot, interleaved):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, x[..., rot:]), dim=-1).half()


def _plain_norm(st):
    c = st["case"]
    angle = st["pos"].double()[st["axis"].long()].t() * st["inv"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    return (_plain_turn(st["q"], st["wq"], cos, sin, c["rot"], c["interleaved"]),
            _plain_turn(st["k"], st["wk"], cos, sin, c["rot"], c["interleaved"]))


def _plain_attn(st):
    c = st["case"]
    hq, hkv, d = c["heads_q"], c["heads_kv"], c["dim"]
    out = torch.empty((st["q"].shape[0], hq, d), dtype=torch.float16, device=DEV)
    iq = ik = 0
    for nq, nk in zip(st["q_lens"], st["k_lens"]):
        k = st["k"][ik:ik + nk].float().permute(1, 2, 0)[:, None]
        v = st["v"][ik:ik + nk].float().permute(1, 0, 2)[:, None]
        step = max(1, (1 << 29) // max(1, hq * nk))
        for r in range(0, nq, step):
            m = min(step, nq - r)
            q = st["q"][iq + r:iq + r + m].float().permute(1, 0, 2).reshape(hkv, hq // hkv, m, d)
            s = (q @ k) * d ** -0.5
            if c["causal"]:
                row = torch.arange(r, r + m, device=DEV)[:, None] + (nk - nq)
                s = s.masked_fill(torch.arange(nk, device=DEV)[None] > row, float("-inf"))
            s = (s - s.amax(-1, keepdim=True)).exp()
            o = (s @ v) / s.sum(-1, keepdim=True)
            out[iq + r:iq + r + m] = o.reshape(hq, m, d).permute(1, 0, 2).half()
        iq, ik = iq + nq, ik + nk
    return out


def run(st):
    op = st["case"]["op"]
    if not own:
        return {"lora": _plain_lora, "norm": _plain_norm, "attn": _plain_attn}[op](st)
    import hopper_gemm_b200 as hg
    if op == "lora":
        return hg.lora(st["X"], st["W"], st["down"], st["up"], st["scale"], st["seg_start"],
                       st["seg_adapter"])
    if op == "norm":
        return hg.qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["pos"], st["inv"], eps=EPS,
                               axis_of=st["axis"] if st["case"]["axes"] > 1 else None,
                               interleaved=st["case"]["interleaved"])
    return hg.attn_prompt(st["q"], st["k"], st["v"], st["cu_q"],
                          st["cu_k"] if st["case"]["past"] else None, causal=st["case"]["causal"])


# ------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "lora":
        x = st["X"].double()
        y = torch.matmul(x, st["W"].double())
        owner = torch.repeat_interleave(torch.tensor(st["ids"], device=DEV),
                                        torch.tensor(st["lens"], device=DEV))
        for a in sorted(set(st["ids"]) - {-1}):
            rows = (owner == a).nonzero().flatten()
            low = x.index_select(0, rows).matmul(st["down"][a].double()) * st["scale"][a].double()
            y.index_add_(0, rows, low.matmul(st["up"][a].double()))
        return y
    if case["op"] == "norm":
        half = case["rot"] // 2
        place = torch.stack([st["pos"][a] for a in st["axis_list"]], dim=1).double()
        unit = torch.polar(torch.ones_like(place), place * st["inv"].double())
        outs = []
        for x, w in ((st["q"], st["wq"]), (st["k"], st["wk"])):
            x = x.double()
            x = x / (x.pow(2).sum(-1, keepdim=True) / case["dim"] + EPS).sqrt() * w.double()
            y = x.clone()
            first = torch.arange(half, device=DEV) * (2 if case["interleaved"] else 1)
            second = first + (1 if case["interleaved"] else half)
            z = torch.complex(x[..., first], x[..., second]) * unit[:, None]
            y[..., first], y[..., second] = z.real, z.imag
            outs.append(y)
        return tuple(outs)
    if case["heads_q"] * _pairs(case) * case["dim"] > 1 << 43:
        return None
    hq, hkv, d = case["heads_q"], case["heads_kv"], case["dim"]
    group = hq // hkv
    cq, ck = _starts(st["q_lens"]), _starts(st["k_lens"])
    y = torch.zeros((cq[-1], hq, d), dtype=torch.float64, device=DEV)
    for b in range(case["batch"]):
        nq, nk = st["q_lens"][b], st["k_lens"][b]
        for h in range(hkv):
            keys = st["k"][ck[b]:ck[b + 1], h].double()
            vals = st["v"][ck[b]:ck[b + 1], h].double()
            for r in range(0, nq, 2048):
                m = min(2048, nq - r)
                last = r + m + nk - nq if case["causal"] else nk
                qs = st["q"][cq[b] + r:cq[b] + r + m, h * group:(h + 1) * group].double()
                z = torch.einsum("qgd,kd->gqk", qs, keys[:last]) / math.sqrt(d)
                if case["causal"]:
                    seen = torch.ones((m, last), dtype=torch.bool, device=DEV).tril(last - m)
                    z = torch.where(seen, z, torch.full_like(z, -math.inf))
                p = torch.softmax(z, dim=-1)
                y[cq[b] + r:cq[b] + r + m, h * group:(h + 1) * group] = \
                    torch.einsum("gqk,kd->qgd", p, vals[:last])
    return y
