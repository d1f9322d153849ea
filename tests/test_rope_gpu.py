"""Rotary positions and the paged append against 64-bit forms: layouts, parts of a head, odd sizes, strides, far positions,
padding, bad pages, other streams, captured graphs."""
import pytest
import torch

from prefix_oracle import PAGE, turn, turn_bound

pytestmark = pytest.mark.gpu


def draw(gen, *shape, dtype=torch.bfloat16):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(0, 1, generator=gen)


@pytest.fixture
def gen(cuda):
    return torch.Generator(device=cuda).manual_seed(7)


def check_turn(got, x, pos, freq, m=1.0, inter=False, inv=False):
    want, w = turn(x, pos, freq, m, inter, inv)
    over = (got.double().cpu() - want).abs() - turn_bound(want, w, x.dtype)
    assert float(over.max()) <= 0, float(over.max())
    dims = 2 * freq.numel()
    assert torch.equal(got[..., dims:], x[..., dims:])


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("rows,heads,D,dims", [(1, 1, 2, 2), (1, 40, 128, 32), (3, 5, 64, 64), (17, 3, 128, 20), (5, 2, 96, 6),
                                               (300, 24, 256, 64), (2, 3, 33, 32), (7, 2, 1024, 1024), (4, 2, 80, 0), (5000, 2, 64, 16)])
def test_rope(gen, rows, heads, D, dims, inter):
    from volundr_mlx_b200 import ops, rotary

    for dtype in (torch.bfloat16, torch.float16):
        x = draw(gen, rows, heads, D, dtype=dtype)
        pos = torch.randint(0, 1 << 20, (rows,), device="cuda", dtype=torch.int32, generator=gen)
        pos[0] = 1 << 28                       # (2^-53 of its turns, 3e-8 of a radian, is inside the bound)
        freq, m = rotary.frequencies(dims, 1e7, scaling="parts", factor=8.0, device="cuda")
        check_turn(ops.rope(x, pos, freq, interleaved=inter, magnitude=m), x, pos, freq, m, inter)
        back = ops.rope(x, pos, freq, interleaved=inter, magnitude=m, inverse=True)
        check_turn(back, x, pos, freq, m, inter, True)
    ops.check_status()


@pytest.mark.parametrize("inter", [False, True])
def test_rope_strides_and_in_place(gen, inter):
    from volundr_mlx_b200 import ops, rotary

    freq, _ = rotary.frequencies(64, 1e4, device="cuda")
    pos = torch.arange(9, device="cuda", dtype=torch.int32) * 1000 - 3000
    for D, off in ((64, 0), (64, 1), (66, 2), (72, 8)):       # 16-byte, odd, 4-byte and 16-byte pieces
        buf = draw(gen, 9, 7 * D + 11)
        x = buf[:, off:off + 5 * D].view(9, 5, D)
        keep = buf.clone()
        out = draw(gen, 5, 9, D).transpose(0, 1)               # heads outermost
        got = ops.rope(x, pos, freq, interleaved=inter, out=out)
        assert got is out
        check_turn(out, x, pos, freq, 1.0, inter)
        assert torch.equal(buf, keep)
        ops.rope(x, pos, freq, interleaved=inter, out=x)       # in place, the rest of the buffer untouched
        assert torch.equal(x, out)
        keep[:, off:off + 5 * D] = buf[:, off:off + 5 * D]
        assert torch.equal(buf, keep)
    e = draw(gen, 1, 1, 64).expand(9, 5, 64)                   # a broadcast input
    check_turn(ops.rope(e, pos, freq, interleaved=inter), e, pos, freq, 1.0, inter)


def test_rope_gradient(gen):
    """The inverse rotation is the gradient: against differences of the 64-bit form, and as the adjoint on the device."""
    from volundr_mlx_b200 import ops, rotary

    freq, m = rotary.frequencies(16, 1e4, scaling="parts", factor=4.0, device="cuda")
    x, g = draw(gen, 3, 2, 24), draw(gen, 3, 2, 24)
    pos = torch.tensor([0, 5, 70000], device="cuda", dtype=torch.int32)
    for inter in (False, True):
        grad = ops.rope(g, pos, freq, interleaved=inter, magnitude=m, inverse=True).double().cpu()
        x64, g64 = x.double().cpu(), g.double().cpu()
        num = torch.zeros_like(x64)
        for i in range(x64.numel()):                            # (linear: any step gives the derivative)
            d = torch.zeros_like(x64).view(-1)
            d[i] = 1.0
            num.view(-1)[i] = ((turn(x64 + d.view_as(x64), pos, freq, m, inter)[0] - turn(x64, pos, freq, m, inter)[0]) * g64).sum()
        w = turn(g64, pos, freq, m, inter, True)[1]
        assert float(((grad - num).abs() - turn_bound(num, w, torch.bfloat16) - 1e-9).max()) <= 0


def append_case(gen, rows, KVH, D, H, dtype, pages=40):
    K, V = draw(gen, pages, KVH, PAGE, D, dtype=dtype), draw(gen, pages, KVH, PAGE, D, dtype=dtype)
    k, v, q = (draw(gen, rows, n, D, dtype=dtype) for n in (KVH, KVH, H))
    return K, V, k, v, q


def want_append(K, V, k, v, table, pos, slot, seq, freq, m, inter):
    wk, w = turn(k, pos, freq, m, inter)
    b = turn_bound(wk, w, k.dtype)
    EK, EV, B = K.double().cpu(), V.clone(), torch.zeros(K.shape, dtype=torch.float64)
    for r in range(k.shape[0]):
        s = int(slot[r])
        if s >= 0:
            page = int(table[int(seq[r]), s // PAGE])
            EK[page, :, s % PAGE], B[page, :, s % PAGE], EV[page, :, s % PAGE] = wk[r], b[r], v[r]
    return EK, B, EV


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,H,KVH,D,dims,inter,T", [(1, 1, 1, 64, 64, False, 1), (5, 40, 8, 128, 32, False, 1), (40, 6, 2, 64, 64, True, 8),
                                                     (130, 3, 3, 128, 128, True, 65), (9, 2, 1, 20, 10, False, 3), (7, 2, 2, 33, 2, True, 7),
                                                     (200, 8, 2, 256, 64, False, 100), (6, 4, 2, 64, 0, False, 2)])
def test_append(gen, rows, H, KVH, D, dims, inter, T, dtype):
    from volundr_mlx_b200 import ops, rotary

    K, V, k, v, q = append_case(gen, rows, KVH, D, H, dtype)
    S = -(-rows // T)
    table = torch.randperm(40, device="cuda", generator=gen).to(torch.int32)[: S * 4].view(S, 4) if S * 4 <= 40 else None
    if table is None:
        S, table = 5, torch.randperm(40, device="cuda", generator=gen).to(torch.int32)[:20].view(5, 4).contiguous()
    r = torch.arange(rows, device="cuda")
    seq = (r % S).int()
    slot = (60 + r // S).int()                                  # crosses a page's end
    slot[-1] = -1 if rows > 1 else 0
    pos = (slot + 100000).int()
    freq, m = rotary.frequencies(dims, 1e7, scaling="ntk", factor=4.0, device="cuda")
    k0, v0, q0, K0, V0 = (t.clone() for t in (k, v, q, K, V))
    q_out = torch.full_like(q, 3.0)
    got = ops.kv_append(k, v, K, V, table, pos, freq if dims else None, slot=slot, seq=seq, q=q, q_out=q_out, interleaved=inter, magnitude=m)
    ops.check_status()
    assert got is q_out and torch.equal(k, k0) and torch.equal(v, v0) and torch.equal(q, q0)
    EK, B, EV = want_append(K0, V0, k, v, table.cpu(), pos, slot, seq, freq, m, inter)
    assert torch.equal(V, EV)
    assert float(((K.double().cpu() - EK).abs() - B).max()) <= 0
    live = rows - (1 if rows > 1 else 0)
    check_turn(q_out[:live], q[:live], pos[:live], freq, m, inter)
    assert bool((q_out[live:] == 3.0).all()), "a padded row's queries were written"
    # without queries, and with the slot and sequence left to their defaults (position, row)
    if rows <= S:
        K2, V2 = K0.clone(), V0.clone()
        assert ops.kv_append(k, v, K2, V2, table, slot, freq, interleaved=inter, magnitude=m) is None
        EK, B, EV = want_append(K0, V0, k, v, table.cpu(), slot, slot, r, freq, m, inter)
        assert torch.equal(V2, EV) and float(((K2.double().cpu() - EK).abs() - B).max()) <= 0


def test_append_bad_pages_are_reported_and_skipped(gen):
    from volundr_mlx_b200 import ops, rotary

    K, V, k, v, _ = append_case(gen, 4, 2, 64, 1, torch.bfloat16, pages=3)
    freq, _ = rotary.frequencies(64, 1e4, device="cuda")
    K0, V0 = K.clone(), V.clone()
    for table, slot, seq in (([[3, 0]], [0] * 4, [0] * 4), ([[-1, 0]], [5] * 4, [0] * 4), ([[1, 0]], [128] * 4, [0] * 4),
                             ([[1, 0]], [3] * 4, [1] * 4), ([[1, 0]], [3] * 4, [-1] * 4)):
        t, s, b = (torch.tensor(x, device="cuda", dtype=torch.int32) for x in (table, slot, seq))
        ops.kv_append(k, v, K, V, t, s, freq, slot=s, seq=b)
        with pytest.raises(RuntimeError, match="index outside"):
            ops.check_status()
        assert torch.equal(K, K0) and torch.equal(V, V0)


def test_append_in_a_graph_follows_its_slots(gen):
    from volundr_mlx_b200 import ops, rotary

    K, V, k, v, q = append_case(gen, 3, 2, 128, 4, torch.bfloat16)
    table = torch.arange(30, device="cuda", dtype=torch.int32).view(3, 10)
    freq, m = rotary.frequencies(128, 1e4, device="cuda")
    slot = torch.zeros(3, device="cuda", dtype=torch.int32)
    pos = torch.zeros_like(slot)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    q_out = torch.zeros_like(q)
    with torch.cuda.graph(g, stream=s):
        ops.kv_append(k, v, K, V, table, pos, freq, slot=slot, q=q, q_out=q_out)
        slot.add_(1)
        pos.add_(1)
    slot.fill_(62)
    pos.fill_(1062)
    K1, V1 = K.clone(), V.clone()
    for _ in range(4):
        g.replay()
    q1 = torch.zeros_like(q)
    for i in range(4):
        sl = torch.full((3,), 62 + i, device="cuda", dtype=torch.int32)
        ops.kv_append(k, v, K1, V1, table, sl + 1000, freq, slot=sl, q=q, q_out=q1)
    assert torch.equal(K, K1) and torch.equal(V, V1) and torch.equal(q_out, q1)
    ops.check_status()


def test_no_rows(gen):
    from volundr_mlx_b200 import ops, rotary

    freq, _ = rotary.frequencies(64, 1e4, device="cuda")
    none = torch.zeros(0, device="cuda", dtype=torch.int32)
    assert ops.rope(draw(gen, 0, 3, 64), none, freq).shape == (0, 3, 64)
    K, V, k, v, _ = append_case(gen, 0, 2, 64, 1, torch.bfloat16)
    assert ops.kv_append(k, v, K, V, torch.zeros((1, 1), device="cuda", dtype=torch.int32), none, freq) is None
