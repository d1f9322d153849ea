"""What is measured of three operators of a decode step over a paged cache whose sequences share a prompt prefix:

rope            rotary positions of [rows, heads, D] activations: half and interleaved layouts, the first `dims` of a head's
                elements, frequencies scaled for long contexts;
kv_append       keys and values of new tokens into their sequences' pages, the keys rotated on the way, and the queries of
                the same tokens rotated in the same pass;
attend_prefix   attention of every sequence's newest token (or newest T tokens) over one prefix that all sequences share
                and the sequence's own pages behind it.

Pages hold 64 tokens: K, V [pages, kv heads, 64, D]. Head counts 40 / 8 (D = 128) are the 32B-shaped model's, 24 heads of
256 with a quarter rotated the reference's defaults, 8 / 2 the two-layer block's; the others are generic."""
import math
import random

import torch

own = False

PAGE = 64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one decode step of sixteen sequences, a quarter of every head rotated
        dict(name="rope_decode", op="rope", rows=16, heads=40, D=128, dims=32, interleaved=False, scaling="none", factor=1.0,
             far=20000, inverse=False, strided=False, type="bf16"),
        # the reference's head shape, an odd number of prompt tokens, turned back (the gradient's direction)
        dict(name="rope_back", op="rope", rows=1999, heads=24, D=256, dims=64, interleaved=False, scaling="linear", factor=4.0,
             far=131072, inverse=True, strided=False, type="fp16"),
        # a long prompt, queries inside a fused projection, frequencies scaled by parts for eight times the context
        dict(name="rope_prompt", op="rope", rows=16384, heads=40, D=128, dims=128, interleaved=True, scaling="parts", factor=8.0,
             far=262144, inverse=False, strided=True, type="bf16"),
        # one decode step: one token for each of thirteen sequences, three padded rows behind them
        dict(name="append_decode", op="append", rows=16, live=13, T=1, heads=40, kv=8, D=128, dims=32, interleaved=False,
             scaling="none", factor=1.0, far=20000, strided=True, type="bf16"),
        # a verify window: eight tokens for each of sixteen sequences, small heads
        dict(name="append_verify", op="append", rows=128, live=128, T=8, heads=32, kv=8, D=64, dims=64, interleaved=True,
             scaling="ntk", factor=4.0, far=65536, strided=True, type="fp16"),
        # prompt chunks of four sequences, 16380 tokens in all
        dict(name="append_prompt", op="append", rows=16380, live=16380, T=4095, heads=40, kv=8, D=128, dims=128,
             interleaved=False, scaling="parts", factor=8.0, far=131072, strided=True, type="bf16"),
        # two young conversations on a short system prompt: the time of the launches
        dict(name="attend_few", op="attend", seqs=2, live=2, T=1, heads=8, kv=2, D=128, prefix=500, lo=1, hi=40, gate=False,
             strided=False, type="bf16"),
        # the decode batch of sixteen (three rows padded) behind a shared document, gated as the model's layers are
        dict(name="attend_batch", op="attend", seqs=16, live=13, T=1, heads=40, kv=8, D=128, prefix=20000, lo=256, hi=2000,
             gate=True, strided=True, type="bf16"),
        # a verify window of eight tokens each, small heads, a prefix that ends inside a page
        dict(name="attend_verify", op="attend", seqs=16, live=16, T=8, heads=32, kv=8, D=64, prefix=8191, lo=9, hi=600,
             gate=False, strided=True, type="fp16"),
        # little is shared, the sequences themselves are long
        dict(name="attend_own", op="attend", seqs=6, live=6, T=1, heads=40, kv=8, D=128, prefix=700, lo=2000, hi=20000,
             gate=False, strided=False, type="bf16"),
        # many samples of one long prompt
        dict(name="attend_many", op="attend", seqs=128, live=128, T=1, heads=40, kv=8, D=128, prefix=32768, lo=16, hi=1024,
             gate=False, strided=False, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["rope", "append", "attend", "attend"])
    t = rng.choice(["bf16", "bf16", "fp16"])
    if op == "attend":
        heads, kv = rng.choice([(40, 8), (40, 8), (8, 2), (32, 8), (16, 16), (12, 2), (24, 1)])
        lo = _log(rng, 1, 2000)
        seqs = _log(rng, 1, 128)
        return dict(op=op, seqs=seqs, live=max(1, seqs - rng.choice([0, 0, 1, 3])), T=rng.choice([1, 1, 1, 2, 5, 8]), heads=heads,
                    kv=kv, D=rng.choice([128, 128, 64]), prefix=_log(rng, 64, 32768), lo=lo, hi=_log(rng, lo, 20000),
                    gate=rng.random() < 0.3, strided=rng.random() < 0.5, type=t)
    D = rng.choice([64, 128, 128, 256])
    dims = rng.choice([D, D, D // 2, D // 4, 20])
    case = dict(op=op, D=D, dims=dims, interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "ntk", "parts"]),
                factor=rng.choice([2.0, 4.0, 8.0]), far=_log(rng, 1000, 1 << 20), strided=rng.random() < 0.5, type=t)
    if op == "rope":
        return dict(case, rows=_log(rng, 1, 16384), heads=rng.choice([1, 2, 8, 24, 40]), inverse=rng.random() < 0.3)
    heads, kv = rng.choice([(40, 8), (8, 2), (32, 8), (16, 16), (12, 2), (24, 1)])
    T = _log(rng, 1, 4095)
    seqs = _log(rng, 1, max(1, min(128, 16380 // T)))
    rows = T * seqs
    return dict(case, rows=rows, live=rows - (T if seqs > 1 and rng.random() < 0.3 else 0), T=T, heads=heads, kv=kv)


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        b, f = most.get(c["op"], (0, 0))
        most[c["op"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        c = _draw(rng)
        w = work(c)
        pool = 2 * c["live"] * c["hi"] * c["kv"] * c["D"] * 2 if c["op"] == "attend" else 0   # (padded to the longest)
        if w["bytes"] <= most[c["op"]][0] and w["flops"] <= most[c["op"]][1] and pool <= 2 << 30:
            return c


def _own_lengths(case):
    """Own tokens of every live sequence, spread evenly over the logarithm of [lo, hi]: the case alone fixes them."""
    n = case["live"]
    r = math.log(case["hi"] / case["lo"])
    return [min(case["hi"], max(case["lo"], round(case["lo"] * math.exp(r * (i / (n - 1) if n > 1 else 1.0))))) for i in range(n)]


def _rows_lengths(case):
    """Own keys that every live row sees: the T newest tokens of a sequence see one more each."""
    T = case["T"]
    return [[max(0, n - T + 1 + t) for t in range(T)] for n in _own_lengths(case)]


def work(case):
    op, D = case["op"], case["D"]
    if op == "rope":
        n = case["rows"] * case["heads"]
        return {"bytes": n * D * 2 * 2 + case["rows"] * 4 + case["dims"] * 4, "flops": n * case["dims"] * 3}
    if op == "append":
        n = case["live"] * (case["heads"] + 2 * case["kv"])
        return {"bytes": n * D * 2 * 2 + case["rows"] * 8 + case["dims"] * 4,
                "flops": case["live"] * (case["heads"] + case["kv"]) * case["dims"] * 3}
    lens = _rows_lengths(case)
    rows = case["live"] * case["T"]
    keys = case["prefix"] + sum(max(x) for x in lens)
    pairs = sum(case["prefix"] + n for x in lens for n in x)
    q = rows * case["heads"] * D * 2
    return {"bytes": keys * case["kv"] * D * 2 * 2 + (3 if case["gate"] else 2) * q, "flops": pairs * case["heads"] * D * 4}


def _frequencies(case):
    """Rotary frequencies in 64 bits: theta^(-2i / dims); `linear` divides them all, `ntk` stretches theta, `parts` divides
    those whose wavelength is long against the trained context and keeps the short ones, with a ramp between."""
    dims, s = case["dims"], case["factor"]
    theta = 1e7
    if case["scaling"] == "ntk" and dims > 2:
        theta *= s ** (dims / (dims - 2))
    f = theta ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    if case["scaling"] == "linear":
        f = f / s
    if case["scaling"] == "parts":
        turns = 4096 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        f = f * (keep + (1 - keep) / s)
    return f, (0.1 * math.log(s) + 1.0 if case["scaling"] == "parts" else 1.0)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    rng = random.Random(seed)
    dt, D = TYPES[case["type"]], case["D"]

    def normal(*shape, std=1.0):
        return torch.empty(shape, dtype=dt, device=dev).normal_(0, std, generator=gen)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    s = {"case": case}
    if case["op"] in ("rope", "append"):
        f, s["magnitude"] = _frequencies(case)
        s["freq"] = f.to(dev)
    if case["op"] == "rope":
        n, H = case["rows"], case["heads"]
        # strided: the queries of a fused projection [q | gate | k | v]
        s["x"] = normal(n, 2 * H + 4, D)[:, :H] if case["strided"] else normal(n, H, D)
        start = rng.randrange(0, max(1, case["far"] - n))
        s["pos"] = (torch.arange(n, device=dev, dtype=torch.int32) + start if n > 64
                    else ints([rng.randrange(case["far"]) for _ in range(n)]))
        s["out"] = torch.zeros((n, H, D), dtype=dt, device=dev)
        return s
    if case["op"] == "append":
        n, T, H, KVH, live = case["rows"], case["T"], case["heads"], case["kv"], case["live"]
        if case["strided"]:
            p = normal(n, H + 2 * KVH, D)
            s["q"], s["k"], s["v"] = p[:, :H], p[:, H:H + KVH], p[:, H + KVH:]
        else:
            s["q"], s["k"], s["v"] = normal(n, H, D), normal(n, KVH, D), normal(n, KVH, D)
        seqs = n // T
        # a sequence's own tokens begin at an odd place of its first page; the shared prefix lies in front of them
        first = [rng.randrange(0, 200) for _ in range(seqs)]
        per = (199 + T + PAGE - 1) // PAGE
        pages = seqs * per + 3
        perm = list(range(pages))
        rng.shuffle(perm)
        s["table"] = ints(perm[:seqs * per]).view(seqs, per)
        b, t = torch.arange(n, device=dev) // T, torch.arange(n, device=dev) % T
        prefix = rng.randrange(0, max(1, case["far"] - 199 - T))
        slot = ints(first)[b] + t.int()
        s["pos"] = (slot + prefix).int()
        slot[live:] = -1
        s["slot"], s["seq"] = slot, b.int()
        s["K"], s["V"] = normal(pages, KVH, PAGE, D), normal(pages, KVH, PAGE, D)
        s["q_out"] = torch.zeros((n, H, D), dtype=dt, device=dev)
        return s
    S, T, H, KVH, live, P = case["seqs"], case["T"], case["heads"], case["kv"], case["live"], case["prefix"]
    lens = _rows_lengths(case)
    rng.shuffle(lens)
    lens += [[-1] * T] * (S - live)
    npre, per = (P + PAGE - 1) // PAGE, max(1, (max(max(x) for x in lens) + PAGE - 1) // PAGE)
    used = [(max(x) + PAGE - 1) // PAGE if max(x) > 0 else 0 for x in lens]
    pages = npre + sum(used) + 2
    perm = list(range(pages))
    rng.shuffle(perm)
    s["prefix_pages"], s["prefix_len"], s["P"] = ints(perm[:npre]), ints([P]), P
    at, table = npre, []
    for u in used:
        table.append(perm[at:at + u] + [-1] * (per - u))
        at += u
    s["table"], s["lens"] = ints(table), ints(lens).view(-1)
    if case["strided"]:   # [q | gate | k | v] rows of a fused projection
        p = normal(S * T, 2 * H + 2 * KVH, D)
        s["q"], s["gate"] = p[:, :H], p[:, H:2 * H]
    else:
        s["q"], s["gate"] = normal(S * T, H, D), normal(S * T, H, D)
    s["q"].mul_(2.0)   # scores of standard deviation two: some keys matter, most do not
    if not case["gate"]:
        s["gate"] = None
    s["K"], s["V"] = normal(pages, KVH, PAGE, D), normal(pages, KVH, PAGE, D)
    s["out"] = torch.zeros((S * T, H, D), dtype=dt, device=dev)
    return s


def _turn(x, pos, freq, magnitude, interleaved, inverse=False):
    """The first 2 * len(freq) elements of every head turned by pos * freq, in 32 bits (the angles in 64)."""
    dims = 2 * freq.numel()
    a = pos.double()[:, None] * freq
    c, s = (torch.cos(a) * magnitude).float()[:, None], (torch.sin(a) * magnitude).float()[:, None]
    if inverse:
        s = -s
    x = x.float()
    if interleaved:
        u, v = x[..., 0:dims:2], x[..., 1:dims:2]
    else:
        u, v = x[..., :dims // 2], x[..., dims // 2:dims]
    a, b = u * c - v * s, u * s + v * c
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., dims:]), -1)


def run(s):
    case = s["case"]
    if case["op"] == "rope":
        if own:
            from volundr_mlx_b200 import ops
            return ops.rope(s["x"], s["pos"], s["freq"], interleaved=case["interleaved"], magnitude=s["magnitude"],
                            inverse=case["inverse"], out=s["out"])
        return _turn(s["x"], s["pos"], s["freq"], s["magnitude"], case["interleaved"], case["inverse"]).to(s["x"].dtype)
    if case["op"] == "append":
        if own:
            from volundr_mlx_b200 import ops
            ops.kv_append(s["k"], s["v"], s["K"], s["V"], s["table"], s["pos"], s["freq"], slot=s["slot"], seq=s["seq"],
                          q=s["q"], q_out=s["q_out"], interleaved=case["interleaved"], magnitude=s["magnitude"])
            return s["q_out"], s["K"], s["V"]
        n, dt = case["live"], s["k"].dtype       # (padded rows lie behind the live ones)
        pos, slot = s["pos"][:n], s["slot"][:n].long()
        s["q_out"][:n] = _turn(s["q"][:n], pos, s["freq"], s["magnitude"], case["interleaved"]).to(dt)
        page = s["table"][s["seq"][:n].long(), slot // PAGE].long()
        s["K"][page, :, slot % PAGE] = _turn(s["k"][:n], pos, s["freq"], s["magnitude"], case["interleaved"]).to(dt)
        s["V"][page, :, slot % PAGE] = s["v"][:n]
        return s["q_out"], s["K"], s["V"]
    if own:
        from volundr_mlx_b200 import ops
        return ops.attend_prefix(s["q"], s["K"], s["V"], s["prefix_pages"], s["prefix_len"], s["table"], s["lens"],
                                 T=case["T"], gate=s["gate"], out=s["out"])
    S, T, H, KVH, D, P = case["seqs"], case["T"], case["heads"], case["kv"], case["D"], s["P"]
    n, G = case["live"], H // KVH
    R, L = n * T, s["table"].shape[1] * PAGE
    q = s["q"][:R].float() * D ** -0.5
    kp = s["K"][s["prefix_pages"]].float().transpose(0, 1).reshape(KVH, -1, D)[:, :P]
    vp = s["V"][s["prefix_pages"]].float().transpose(0, 1).reshape(KVH, -1, D)[:, :P]
    sp = torch.matmul(q.view(R, KVH, G, D).transpose(0, 1).reshape(KVH, R * G, D), kp.transpose(1, 2))
    sp = sp.view(KVH, n, T * G, P).transpose(0, 1)                                    # [n, KVH, T G, P]
    page = s["table"][:n].clamp(min=0)
    ko = s["K"][page].float().transpose(1, 2).reshape(n, KVH, L, D)
    vo = s["V"][page].float().transpose(1, 2).reshape(n, KVH, L, D)
    so = torch.matmul(q.view(n, T, KVH, G, D).transpose(1, 2).reshape(n, KVH, T * G, D), ko.transpose(2, 3))
    lens = s["lens"][:R].view(n, 1, T, 1).expand(n, 1, T, G).reshape(n, 1, T * G, 1)
    so = so.masked_fill(torch.arange(L, device=q.device) >= lens, -math.inf)
    m = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    ep, eo = torch.exp(sp - m), torch.exp(so - m)
    o = torch.matmul(ep.transpose(0, 1).reshape(KVH, n * T * G, P), vp).view(KVH, n, T * G, D).transpose(0, 1)
    o = (o + torch.matmul(eo, vo)) / (ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True))
    o = o.view(n, KVH, T, G, D).transpose(1, 2).reshape(R, H, D)
    if s["gate"] is not None:
        o = o / (1 + torch.exp(-s["gate"][:R].float()))
    s["out"][:R] = o.to(s["out"].dtype)
    return s["out"]


def _exact_turn(x, pos, freq, magnitude, interleaved, sign):
    """Complex multiplication by magnitude * exp(i sign pos freq), pair by pair, in 64 bits."""
    h = freq.numel()
    y = x.double().clone()
    w = torch.polar(torch.full((pos.numel(), h), float(magnitude), dtype=torch.float64, device=x.device),
                    sign * pos.double()[:, None] * freq[None, :])[:, None, :]
    if interleaved:
        y[..., :2 * h] = torch.view_as_real(torch.view_as_complex(y[..., :2 * h].reshape(*y.shape[:-1], h, 2).contiguous()) * w).flatten(-2)
    else:
        z = torch.complex(y[..., :h].contiguous(), y[..., h:2 * h].contiguous()) * w
        y[..., :h], y[..., h:2 * h] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_turn(s["x"], s["pos"], s["freq"], s["magnitude"], case["interleaved"], -1.0 if case["inverse"] else 1.0)
    if case["op"] == "append":
        n = case["live"]
        q, K, V = s["q_out"].double(), s["K"].double(), s["V"].double()
        q[:n] = _exact_turn(s["q"][:n], s["pos"][:n], s["freq"], s["magnitude"], case["interleaved"], 1.0)
        k = _exact_turn(s["k"][:n], s["pos"][:n], s["freq"], s["magnitude"], case["interleaved"], 1.0)
        at = s["table"].long().gather(1, (s["slot"][:n].long() // PAGE).view(-1, case["T"])).view(-1) * PAGE + s["slot"][:n] % PAGE
        for dst, src in ((K, k), (V, s["v"][:n].double())):
            flat = dst.transpose(1, 2).reshape(-1, case["kv"], case["D"])
            flat[at] = src
            dst.copy_(flat.view(dst.shape[0], PAGE, case["kv"], case["D"]).transpose(1, 2))
        return q, K, V
    # sequence by sequence, kv head by kv head: the keys of prefix and own pages in one list, one softmax
    out = s["out"].double()
    T, D, P = case["T"], case["D"], s["P"]
    G = case["heads"] // case["kv"]
    lens = s["lens"].tolist()
    for h in range(case["kv"]):
        kp = s["K"][s["prefix_pages"], h].double().reshape(-1, D)[:P]
        vp = s["V"][s["prefix_pages"], h].double().reshape(-1, D)[:P]
        for b in range(case["live"]):
            most = max(lens[b * T:(b + 1) * T])
            pages = s["table"][b, :(most + PAGE - 1) // PAGE]
            k = torch.cat((kp, s["K"][pages, h].double().reshape(-1, D)[:most]))
            v = torch.cat((vp, s["V"][pages, h].double().reshape(-1, D)[:most]))
            for t in range(T):
                r, n = b * T + t, P + lens[b * T + t]
                a = torch.softmax(torch.einsum("gd,kd->gk", s["q"][r, h * G:(h + 1) * G].double(), k[:n]) / math.sqrt(D), dim=-1)
                out[r, h * G:(h + 1) * G] = torch.einsum("gk,kd->gd", a, v[:n])
    if s["gate"] is not None:
        live = torch.arange(out.shape[0], device=out.device) < case["live"] * T
        out = torch.where(live[:, None, None], out * torch.sigmoid(s["gate"].double()), out)
    return out
