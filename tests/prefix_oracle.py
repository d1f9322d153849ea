"""Plain 64-bit forms of the rotary, append and shared-prefix attention operators, and their error bounds."""
import torch

PAGE = 64


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def turn(x, pos, freq, magnitude=1.0, interleaved=False, inverse=False):
    """(rotated, |u| + |v| of every element's pair) in 64 bits."""
    x = x.double().cpu()
    h = freq.numel()
    a = pos.double().cpu()[:, None, None] * freq.cpu()
    c, s = torch.cos(a) * magnitude, torch.sin(a) * magnitude * (-1.0 if inverse else 1.0)
    i0 = torch.arange(h) * (2 if interleaved else 1)
    i1 = i0 + (1 if interleaved else h)
    y, w = x.clone(), torch.zeros_like(x)
    y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i0] * s + x[..., i1] * c
    w[..., i0] = w[..., i1] = (x[..., i0].abs() + x[..., i1].abs()) * magnitude
    return y, w


def turn_bound(want, w, dtype):
    """One rounding to the storage type (half a step, also of its smallest numbers) on top of the fp32 error of the pair: the
    angle's fraction 2^-25 turns and the sine's two units give 4e-7 of |u| + |v|, the two products and the sum 2e-7."""
    return half_step(dtype) * want.abs() + 6.1e-7 * w + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def attend(q, K, V, prefix_pages, P, table, lens, T, scale=None, gate=None):
    """(out, bound) in 64 bits, row by row; rows with lens < 0 are None."""
    dtype = q.dtype
    q, K, V = q.double(), K.double(), V.double()
    R, H, D = q.shape
    KVH = K.shape[1]
    G = H // KVH
    scale = D ** -0.5 if scale is None else scale
    u = half_step(dtype)
    out = []
    for r in range(R):
        n = int(lens[r])
        if n < 0:
            out.append(None)
            continue
        npre, nown = (P + PAGE - 1) // PAGE, (n + PAGE - 1) // PAGE
        pages = [int(p) for p in prefix_pages[:npre]], [int(p) for p in table[r // T, :nown]]

        def rows(X):
            return torch.cat([X[pg].transpose(0, 1).reshape(KVH, -1, D)[:, :m] for pg, m in zip(pages, (P, n))], 1)

        k, v = rows(K), rows(V)                                       # [KVH, keys, D]
        if k.shape[1] == 0:
            out.append((torch.zeros((H, D), dtype=torch.float64, device=q.device),) * 2)
            continue
        x = q[r].view(KVH, G, D)
        s = torch.einsum("hgd,hkd->hgk", x, k) * scale
        p = torch.softmax(s, -1)
        o, a = torch.einsum("hgk,hkd->hgd", p, v), torch.einsum("hgk,hkd->hgd", p, v.abs())
        # scores: fp32 sums of D products; probabilities: one rounding to the storage type; fp32 sums over the keys (in
        # blocks of 128 and pieces of them, 2^-24 per addition on the longest chain); the result rounded once
        ds = (D + 16) * 2.0 ** -24 * (torch.einsum("hgd,hkd->hgk", x.abs(), k.abs()) * scale).amax(-1, keepdim=True)
        chain = (k.shape[1] / 16 + 256) * 2.0 ** -24
        b = (u + 2 * ds + 2 * chain) * a * 1.01 + torch.finfo(dtype).smallest_normal
        if gate is not None:
            g = torch.sigmoid(gate[r].double()).view(KVH, G, D)
            o, b = o * g, b * g + 1e-6 * (o * g).abs()
        out.append((o.reshape(H, D), (b + u * (o.abs() + b)).reshape(H, D)))
    return out


def check_attend(got, want, before):
    for r, w in enumerate(want):
        if w is None:
            assert torch.equal(got[r], before[r]), f"padded row {r} was written"
        else:
            over = (got[r].double() - w[0]).abs() - w[1]
            assert not torch.isnan(got[r]).any() and float(over.max()) <= 0, f"row {r}: {float(over.max()):.3e} over its bound"
