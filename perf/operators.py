"""Cases, plain forms and 64-bit values of the serving and rotary operators.

Three operators: ``paged_sdpa`` (attention of new tokens over a paged cache),
``paged_append`` (writing new keys and values into that cache, keys normed and
rotated on the way, queries with them) and ``qk_norm_rope`` (the same norm and
rotation for training, with its gradient).  With ``own`` false, ``run`` computes
them from elementary torch operations in float32; with ``own`` true, it makes the
framework's calls.
"""
import importlib
import math
import random

import torch

own = False

EPS = 1e-6  # of the norms, and of the row sum inside ``stats``
TYPES = {"f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one user's single token over a short context: latency
        dict(name="decode_one", op="attend", type="f16", seqs=1, q_max=1, kv_max=700, mix="even", hq=8, hkv=8, d=64, dv=64,
             page=16, ragged=1),
        # a serving step: 32 users, contexts of every length, grouped heads
        dict(name="decode_batch", op="attend", type="f16", seqs=32, q_max=1, kv_max=8192, mix="ragged", hq=32, hkv=8, d=128,
             dv=128, page=64, ragged=2),
        # long documents, one token each: the cache's bytes
        dict(name="decode_long", op="attend", type="f16", seqs=16, q_max=1, kv_max=32768, mix="even", hq=32, hkv=4, d=128,
             dv=128, page=128, ragged=3),
        # a few drafted tokens a user, every head with keys of its own, fp32
        dict(name="drafts_f32", op="attend", type="f32", seqs=8, q_max=5, kv_max=4096, mix="ragged", hq=16, hkv=16, d=64,
             dv=64, page=32, ragged=4),
        # ragged chunks of several prompts
        dict(name="chunks", op="attend", type="f16", seqs=4, q_max=512, kv_max=8192, mix="ragged", hq=16, hkv=4, d=64, dv=64,
             page=16, ragged=6),
        # two long prompts, a chunk of each: the largest products
        dict(name="chunks_large", op="attend", type="f16", seqs=2, q_max=2048, kv_max=16384, mix="even", hq=32, hkv=8, d=128,
             dv=128, page=64, ragged=6),
        # one prompt's chunk among single tokens of other users
        dict(name="mixed", op="attend", type="f16", seqs=12, q_max=384, kv_max=8192, mix="one", hq=32, hkv=8, d=128, dv=128,
             page=32, ragged=6),
        # the write before a serving step's attention: one token a user
        dict(name="append_tokens", op="append", type="f16", seqs=16, q_max=1, kv_max=2048, mix="ragged", hq=32, hkv=8, d=128,
             dv=128, page=64, ragged=8, rot=128, norm=True, pairs="halves", weight="f16"),
        # the write before a prompt chunk's attention
        dict(name="append_chunks", op="append", type="f16", seqs=5, q_max=2048, kv_max=4096, mix="ragged", hq=32, hkv=8,
             d=128, dv=128, page=16, ragged=9, rot=128, norm=True, pairs="halves", weight="f32"),
        # a short sequence's forward: latency
        dict(name="rope_small", op="rope", type="f16", batch=1, seq=61, hq=8, hk=8, d=64, rot=64, norm=True, pairs="halves",
             weight="f16", grad=False, packed=False),
        # a training step's forward and backward
        dict(name="rope_train", op="rope", type="f16", batch=4, seq=8192, hq=16, hk=16, d=128, rot=128, norm=True,
             pairs="halves", weight="f32", grad=True, packed=False),
        # fp32, packed odd lengths, grouped heads, part of the features rotated in neighbouring pairs
        dict(name="rope_train_f32", op="rope", type="f32", batch=1, seq=4099, hq=12, hk=4, d=64, rot=32, norm=True,
             pairs="neighbours", weight="f32", grad=True, packed=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "chunk", "append", "rope", "rope"])
    dtype = rng.choice(["f16", "f16", "f32"])
    d = rng.choice([64, 128, rng.randrange(2, 17) * 8])
    if kind == "rope":
        hq = _log(rng, 1, 32)
        return dict(op="rope", type=dtype, batch=_log(rng, 1, 4), seq=_log(rng, 1, 8192), hq=min(hq, 16), hk=rng.randint(1, min(hq, 16)),
                    d=d, rot=rng.choice([d, d, rng.randrange(1, d // 8 + 1) * 8]), norm=rng.random() < 0.8,
                    pairs=rng.choice(["halves", "neighbours"]), weight=rng.choice([dtype, "f32"]), grad=rng.random() < 0.6,
                    packed=rng.random() < 0.5)
    hkv = rng.choice([1, 2, 4, 8])
    case = dict(type=dtype, hkv=hkv, hq=hkv * rng.choice([1, 2, 3, 4, 8]), d=d, dv=rng.choice([d, d, rng.randrange(2, 17) * 8]),
                page=rng.choice([16, 32, 64, 128, 256]), ragged=rng.randrange(1, 10 ** 6))
    case["hq"] = min(case["hq"], 32) // hkv * hkv
    if kind == "decode":
        case |= dict(op="attend", seqs=_log(rng, 1, 48), q_max=rng.choice([1, 1, 1, 2, 4, 7]), kv_max=_log(rng, 16, 8192),
                     mix=rng.choice(["even", "ragged"]))
    elif kind == "chunk":
        q_max = _log(rng, 8, 1024)
        case |= dict(op="attend", seqs=_log(rng, 1, 6), q_max=q_max, kv_max=q_max + _log(rng, 1, 4096 if dtype == "f16" else 1024),
                     mix=rng.choice(["even", "ragged", "one"]))
    else:
        q_max = _log(rng, 1, 1024)
        case |= dict(op="append", seqs=_log(rng, 1, 8), q_max=q_max, kv_max=q_max + _log(rng, 1, 2048),
                     mix=rng.choice(["even", "ragged", "one"]), rot=rng.choice([0, d, d, rng.randrange(1, d // 8 + 1) * 8]),
                     norm=rng.random() < 0.6, pairs=rng.choice(["halves", "neighbours"]), weight=rng.choice([dtype, "f32"]))
    return case


def _lengths(case):
    """New tokens and cached tokens (the new ones included) of each sequence."""
    r = random.Random(case["ragged"])
    new, held = [], []
    for n in range(case["seqs"]):
        if case["mix"] == "even":
            a, b = case["q_max"], case["kv_max"]
        elif case["mix"] == "one":
            a = case["q_max"] if n == 0 else 1
            b = max(a, _log(r, max(1, case["kv_max"] // 16), case["kv_max"]))
        else:
            a = r.randint(1, case["q_max"])
            b = max(a, _log(r, max(1, case["kv_max"] // 64), case["kv_max"]))
        new.append(a)
        held.append(max(a, b))
    return new, held


def _table(positions, rot):
    """cos | sin of position * 10000^(-2i/rot), [positions, rot] float32."""
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]

    def normal(*shape, to=dtype):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(to)

    def weight():
        return (1 + 0.1 * torch.randn(case["d"], generator=g, device="cuda")).to(TYPES[case["weight"]])

    s = dict(case=case)
    if case["op"] == "rope":
        b, n, d = case["batch"], case["seq"], case["d"]
        s |= dict(q=normal(b, n, case["hq"], d), k=normal(b, n, case["hk"], d), q_weight=None, k_weight=None, positions=None)
        if case["norm"]:
            s |= dict(q_weight=weight(), k_weight=weight())
        if case["packed"]:  # documents of at most 512 tokens, one behind the other
            s["positions"] = (torch.arange(n, device="cuda", dtype=torch.int32) % 512).expand(b, n).contiguous()
        s["table"] = _table(512 if case["packed"] else n, case["rot"])
        if case["grad"]:
            s["leaves"] = [x.requires_grad_() for x in (s["q"], s["k"], s["q_weight"], s["k_weight"]) if x is not None]
            s["d_out"] = [normal(*s["q"].shape), normal(*s["k"].shape)]
        return s
    new, held = _lengths(case)
    order = random.Random(case["ragged"] + 1)
    page, t = case["page"], sum(new)
    used = [-(-x // page) for x in held]
    pool = sum(used) + 2
    ids = list(range(pool))
    order.shuffle(ids)  # a cache in use: pages of a sequence lie anywhere
    width = max(used)
    rows, at = [], 0
    for u in used:
        rows.append(ids[at:at + u] + [-1] * (width - u))
        at += u
    start = [0]
    for x in new:
        start.append(start[-1] + x)
    s |= dict(page_table=torch.tensor(rows, dtype=torch.int32, device="cuda"),
              kv_len=torch.tensor(held, dtype=torch.int32, device="cuda"),
              q_start=torch.tensor(start, dtype=torch.int32, device="cuda"), q_max=max(new), kv_max=max(held),
              k_pages=normal(pool, page, case["hkv"], case["d"]), v_pages=normal(pool, page, case["hkv"], case["dv"]),
              q=normal(t, case["hq"], case["d"]), scale=case["d"] ** -0.5)
    if case["op"] == "append":
        s |= dict(k=normal(t, case["hkv"], case["d"]), v=normal(t, case["hkv"], case["dv"]), table=None, q_weight=None,
                  k_weight=None)
        if case["rot"]:
            s["table"] = _table(case["kv_max"], case["rot"])
        if case["norm"]:
            s |= dict(q_weight=weight(), k_weight=weight())
    return s


# ------------------------------------------------------------------ plain forms
def _norm(x, weight):
    x = x.float()
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()


def _rotate(x, table, positions, pairs):
    """x [..., heads, d] at positions [...], its first `rot` features rotated."""
    if table is None:
        return x
    half = table.shape[1] // 2
    row = table[positions].unsqueeze(-2)
    cos, sin = row[..., :half], row[..., half:]
    x, rest = x[..., :2 * half], x[..., 2 * half:]
    if pairs == "halves":
        a, b = x[..., :half], x[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0::2], x[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_rope(s):
    pairs, positions = s["case"]["pairs"], s["positions"]
    if positions is None:
        positions = torch.arange(s["q"].shape[1], device="cuda").expand(s["q"].shape[:2])
    return [_rotate(_norm(s[x], s[x + "_weight"]), s["table"], positions, pairs).to(s[x].dtype) for x in ("q", "k")]


def _places(s):
    """Sequence, place among its new tokens and position of each new token."""
    q_start = s["q_start"].long()
    t = torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(q_start[1:].contiguous(), t, right=True)
    place = t - q_start[seq]
    return seq, place, s["kv_len"].long()[seq] - (q_start[seq + 1] - q_start[seq]) + place


def _plain_append(s):
    seq, _, at = _places(s)
    page = s["k_pages"].shape[1]
    where = (s["page_table"][seq, at // page].long(), at % page)
    pairs, dtype = s["case"]["pairs"], s["k"].dtype
    s["k_pages"][where] = _rotate(_norm(s["k"], s["k_weight"]), s["table"], at, pairs).to(dtype)
    s["v_pages"][where] = s["v"]
    return _rotate(_norm(s["q"], s["q_weight"]), s["table"], at, pairs).to(dtype), s["k_pages"], s["v_pages"]


def _plain_attend(s):
    q, kv_len, q_start = s["q"], s["kv_len"].long(), s["q_start"].long()
    q_max, kv_max, (_, page, hkv, d), dv = s["q_max"], s["kv_max"], s["k_pages"].shape, s["v_pages"].shape[3]
    n, group = kv_len.shape[0], q.shape[1] // hkv
    i = torch.arange(q_max, device="cuda")
    j = torch.arange(kv_max, device="cuda")
    new = q_start[1:] - q_start[:-1]
    tokens = (q_start[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qs = q[tokens].float().view(n, q_max, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, group * q_max, d)
    pages = s["page_table"][:, :-(-kv_max // page)].long()
    ks = s["k_pages"][pages].flatten(1, 2)[:, :kv_max].transpose(1, 2).float()
    vs = s["v_pages"][pages].flatten(1, 2)[:, :kv_max].transpose(1, 2).float()
    seen = j < ((kv_len - new)[:, None] + i + 1)[..., None]  # [n, q_max, kv_max]
    x = (qs @ ks.transpose(2, 3)).mul_(s["scale"]).view(n, hkv, group, q_max, kv_max)
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(n, hkv, group * q_max, kv_max) @ vs).view(n, hkv, group, q_max, dv) / total
    stats = (top + torch.log(total + EPS)).squeeze(-1)
    seq, place, _ = _places(s)
    return o[seq, :, :, place].reshape(-1, hkv * group, dv).to(q.dtype), stats[seq, :, :, place].reshape(-1, hkv * group)


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    fa = importlib.import_module("tf-custom-flash-attention_b200")
    case = s["case"]
    if case["op"] == "attend":
        return fa.paged_sdpa(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_len"], s["q_start"], scale=s["scale"])
    interleaved = case["pairs"] == "neighbours"
    if case["op"] == "append":
        q = fa.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_len"], s["q_start"], q=s["q"],
                            q_weight=s["q_weight"], k_weight=s["k_weight"], table=s["table"], eps=EPS, interleaved=interleaved)
        return q, s["k_pages"], s["v_pages"]
    call = fa.autograd.qk_norm_rope if case["grad"] else fa.qk_norm_rope
    return call(s["q"], s["k"], s["q_weight"], s["k_weight"], s["table"], s["positions"], eps=EPS, interleaved=interleaved)


def run(state):
    if own:
        outs = _own(state)
    else:
        outs = {"attend": _plain_attend, "append": _plain_append, "rope": _plain_rope}[state["case"]["op"]](state)
    if state["case"].get("grad"):
        return [x.detach() for x in outs] + list(torch.autograd.grad(outs, state["leaves"], state["d_out"]))
    return list(outs)


def work(case):
    size = 2 if case["type"] == "f16" else 4
    if case["op"] == "rope":
        rows = case["batch"] * case["seq"] * (case["hq"] + case["hk"])
        if case["grad"]:  # x and its output; x again, the output's gradient and x's
            return {"bytes": 4 * rows * case["d"] * size, "flops": rows * case["d"] * 22}
        return {"bytes": 2 * rows * case["d"] * size, "flops": rows * case["d"] * 8}
    new, held = _lengths(case)
    t, hq, hkv, d, dv = sum(new), case["hq"], case["hkv"], case["d"], case["dv"]
    if case["op"] == "append":
        return {"bytes": 2 * t * (hq * d + hkv * (d + dv)) * size, "flops": t * (hq + hkv) * d * 8}
    seen = sum(a * (b - a) + a * (a + 1) // 2 for a, b in zip(new, held))
    return {"bytes": t * hq * ((d + dv) * size + 4) + sum(held) * hkv * (d + dv) * size, "flops": 2 * seen * hq * (d + dv)}


# ------------------------------------------------------------------ 64 bits
def _exact_turn(x, weight, angles, pairs):
    """One tensor [tokens, heads, d] in float64: norm by the weight, then a rotation by angles [tokens, rot / 2]."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / y.shape[-1] + EPS) * weight.double()
    if angles is None:
        return y
    h = angles.shape[1]
    first = torch.arange(h, device="cuda") * (1 if pairs == "halves" else 2)
    second = first + (h if pairs == "halves" else 1)
    turn = torch.polar(torch.ones_like(angles), angles)[:, None]
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
    out = y.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _angles(positions, table):
    """The angles whose cosines and sines the (float32) table holds."""
    if table is None:
        return None
    h = table.shape[1] // 2
    return positions.double()[:, None] * 10000.0 ** (-torch.arange(h, dtype=torch.float64, device="cuda") / h)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        b, n = s["q"].shape[:2]
        pos = torch.arange(n, device="cuda").repeat(b) if s["positions"] is None else s["positions"].reshape(-1)
        a = _angles(pos, s["table"])
        outs, grads, weights = [], [], []
        for x in ("q", "k"):
            w = s[x + "_weight"]
            y = s[x].detach().double().flatten(0, 1).requires_grad_(case["grad"])
            w = w if w is None else w.detach().double().requires_grad_(case["grad"])
            z = _exact_turn(y, w, a, case["pairs"])
            outs.append(z.detach().view(s[x].shape))
            if case["grad"]:
                got = torch.autograd.grad(z, [y] if w is None else [y, w], s["d_out"][len(grads)].double().flatten(0, 1))
                grads.append(got[0].view(s[x].shape))
                weights += got[1:]
        return outs + grads + weights
    start, held = s["q_start"].tolist(), s["kv_len"].tolist()
    page, group = case["page"], case["hq"] // case["hkv"]
    if case["op"] == "append":
        q = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        for n, kv in enumerate(held):
            a, e = start[n], start[n + 1]
            pos = torch.arange(kv - (e - a), kv, device="cuda")
            ang = _angles(pos, s["table"])
            slots = s["page_table"][n].long()[pos // page] * page + pos % page
            q[a:e] = _exact_turn(s["q"][a:e], s["q_weight"], ang, case["pairs"])
            kp.flatten(0, 1)[slots] = _exact_turn(s["k"][a:e], s["k_weight"], ang, case["pairs"])
            vp.flatten(0, 1)[slots] = s["v"][a:e].double()
        return [q, kp, vp]
    out = torch.empty(*s["q"].shape[:2], case["dv"], dtype=torch.float64, device="cuda")
    stats = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for n, kv in enumerate(held):
        a, e = start[n], start[n + 1]
        pos = torch.arange(kv, device="cuda")
        slots = s["page_table"][n].long()[pos // page] * page + pos % page
        hidden = pos[None] > torch.arange(kv - (e - a), kv, device="cuda")[:, None]
        for h in range(case["hq"]):
            k = s["k_pages"].flatten(0, 1)[slots, h // group].double()
            x = (s["q"][a:e, h].double() @ k.T * s["scale"]).masked_fill(hidden, -math.inf)
            out[a:e, h] = torch.softmax(x, -1) @ s["v_pages"].flatten(0, 1)[slots, h // group].double()
            m = x.max(-1).values
            stats[a:e, h] = m + torch.log(torch.exp(x - m[:, None]).sum(-1) + EPS)
    return [out, stats]
