"""Attention over a shared prefix against a 64-bit softmax: lengths around page and block edges, empty rows, padded rows, head
layouts from one query head per kv head to more than a tile, windows, strides, gates, anything in the invisible places."""
import math

import pytest
import torch

from prefix_oracle import PAGE, attend, check_attend

pytestmark = pytest.mark.gpu


class Case:
    """A pool whose invisible places hold NaN and infinities, tables whose unused entries are no pages."""

    def __init__(self, H, KVH, D, P, lens, T=1, dtype=torch.bfloat16, gate=False, strided=False, seed=0, spread=2.0, spare=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape):
            return torch.empty(shape, device="cuda", dtype=dtype).normal_(0, 1, generator=gen)

        self.T, self.P, self.H, self.D = T, P, H, D
        R, S = len(lens), len(lens) // T
        own = [max(0, max(lens[b * T:(b + 1) * T])) for b in range(S)]
        npre, need = -(-P // PAGE), [-(-n // PAGE) for n in own]
        pages = npre + sum(need) + 2
        perm = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
        self.prefix_pages = torch.cat([perm[:npre], torch.full((spare,), -7, device="cuda", dtype=torch.int32)])
        self.table = torch.full((S, max(need + [0]) + spare), -1, device="cuda", dtype=torch.int32)
        vis = torch.zeros((pages, PAGE), dtype=torch.bool, device="cuda")

        def see(ids, n):
            for i, p in enumerate(ids.tolist()):
                vis[p, : min(PAGE, n - i * PAGE)] = True

        see(perm[:npre], P)
        at = npre
        for b in range(S):
            self.table[b, : need[b]] = perm[at: at + need[b]]
            see(perm[at: at + need[b]], own[b])
            at += need[b]
        self.K, self.V = normal(pages, KVH, PAGE, D), normal(pages, KVH, PAGE, D)
        hidden = ~vis[:, None, :, None].expand_as(self.K)
        bad = torch.tensor([math.nan, math.inf, -math.inf], device="cuda", dtype=dtype)
        self.K[hidden] = bad[torch.arange(int(hidden.sum()), device="cuda") % 3]
        self.V[hidden] = bad[torch.arange(int(hidden.sum()), device="cuda") % 3]
        p = normal(R, 2 * H + 3, D)
        self.q = (p[:, :H] if strided else normal(R, H, D))
        self.q.mul_(spread)
        self.gate = None if not gate else (p[:, H:2 * H] if strided else normal(R, H, D))
        self.lens = torch.tensor(lens, device="cuda", dtype=torch.int32)
        self.prefix_len = torch.tensor([P], device="cuda", dtype=torch.int32)
        buf = torch.full((R, H + 1, D), 5.0, device="cuda", dtype=dtype)
        self.out = buf[:, :H] if strided else buf[:, :H].contiguous()

    def run(self, **kw):
        from volundr_mlx_b200 import ops

        return ops.attend_prefix(self.q, self.K, self.V, self.prefix_pages, self.prefix_len, self.table, self.lens, T=self.T,
                                 **{"gate": self.gate, "out": self.out, **kw})

    def want(self, **kw):
        return attend(self.q, self.K, self.V, self.prefix_pages, self.P, self.table, self.lens, self.T, gate=self.gate, **kw)

    def check(self, **kw):
        from volundr_mlx_b200 import ops

        before = self.out.clone()
        got = self.run(**kw)
        ops.check_status()
        assert got is self.out
        check_attend(got, self.want(**kw), before)


EDGES = [0, 1, 2, 63, 64, 65, 127, 128, 129, 191, 192, 193, 256, 257, 700]


@pytest.mark.parametrize("P", [0, 1, 63, 64, 65, 128, 129, 500, 1025])
def test_lengths(cuda, P):
    Case(5, 1, 128, P, EDGES, seed=P, spare=2).check()


@pytest.mark.parametrize("P", [0, 1, 64, 129, 1000])
def test_lengths_small_heads(cuda, P):
    Case(4, 2, 64, P, EDGES[::-1], dtype=torch.float16, seed=P).check()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,KVH,S", [(1, 1, 1), (1, 1, 40), (16, 16, 3), (6, 1, 21), (6, 1, 22), (24, 1, 11), (40, 8, 16), (128, 1, 2),
                                     (129, 1, 3), (8, 2, 70), (130, 1, 5)])
def test_head_layouts(cuda, H, KVH, S, D):
    Case(H, KVH, D, 333, [(37 * i) % 150 for i in range(S)], dtype=[torch.bfloat16, torch.float16][S % 2], seed=H + S).check()


@pytest.mark.parametrize("H,KVH,D,T,P", [(40, 8, 128, 8, 500), (24, 1, 64, 8, 129), (5, 1, 128, 60, 64), (2, 2, 64, 3, 0), (8, 2, 128, 2, 1)])
def test_windows(cuda, H, KVH, D, T, P):
    """T newest tokens of a sequence see one key more each; a sequence younger than the window; a padded sequence."""
    lens = []
    for n in (T, T + 5, 130, 64, 700):
        lens += [max(0, n - T + 1 + t) for t in range(T)]
    lens += [-1] * T
    Case(H, KVH, D, P, lens, T=T, seed=T, strided=True).check()


@pytest.mark.parametrize("lens,P", [([-1, 3, -1, 0, 64, -1], 100), ([-1, -1], 100), ([0, 0, 0], 0), ([0, -1, 5], 0), ([-1] * 5 + [1], 64)])
def test_padded_and_empty_rows(cuda, lens, P):
    Case(6, 2, 64, P, lens, seed=3, strided=True).check()
    Case(10, 2, 128, P, lens, seed=3, gate=True).check()


def test_mixed_rows_of_a_window(cuda):
    """Padded rows inside a window, rows that see nothing beside rows that see much."""
    Case(4, 2, 128, 70, [-1, 3, 200, 0, -1, 65, 1, 130, -1], T=3, seed=9).check()
    Case(4, 2, 128, 0, [-1, 3, 200, 0, -1, 65, 1, 130, -1], T=3, seed=9).check()


@pytest.mark.parametrize("strided", [False, True])
def test_gate_scale_and_strides(cuda, strided):
    c = Case(10, 2, 128, 200, [3, 77, 500], gate=True, strided=strided, seed=5)
    c.check()
    c.check(scale=0.3)


def test_sharp_and_flat_scores(cuda):
    """Scores of standard deviation 40 (one key takes all, the running maximum jumps) and all-equal scores."""
    Case(8, 2, 128, 900, [10, 300, 0], seed=6, spread=40.0).check()
    Case(8, 2, 128, 900, [10, 300, 0], seed=6, spread=0.0).check()
    c = Case(8, 2, 64, 900, [10, 300, 0], seed=6, dtype=torch.float16)
    c.q.abs_()
    ramp = torch.arange(c.K.shape[0] * PAGE, device=c.K.device).view(-1, 1, PAGE, 1) / (c.K.shape[0] * PAGE) * 4
    fin = torch.isfinite(c.K)
    c.K.copy_(torch.where(fin, ramp.to(c.K.dtype).expand_as(c.K), c.K))     # scores that grow from page to page
    c.check()
    c.q.neg_()
    c.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,KVH", [(40, 2), (2, 2)])
def test_one_key_far_above_many(cuda, dtype, H, KVH):
    """One key of the prefix takes as much as thousands of small ones together: their probabilities are 2^-14 and less of the
    largest, where fp16 without a common factor has lost most of its bits."""
    c = Case(H, KVH, 64, 9000, [1000, 5, 0, 64], seed=22, dtype=dtype, spread=0.0)
    c.q.fill_(0.5)
    fin = torch.isfinite(c.K)
    c.K.copy_(torch.where(fin, torch.zeros_like(c.K), c.K))
    c.K[int(c.prefix_pages[3]), :, 17] = 2.5            # score 64 * 0.5 * 2.5 / 8 = 10: e^-10 = 4.5e-5 = 2^-14.4
    c.check()


def test_long_prefix_and_long_own(cuda):
    Case(10, 2, 128, 20011, [1, 4000, 17], seed=11).check()
    Case(16, 16, 64, 130, [9000, 3, 12345], seed=12).check()


def test_many_rows(cuda):
    Case(40, 8, 128, 1500, [(13 * i) % 97 for i in range(128)], seed=13).check()


@pytest.mark.parametrize("D,T", [(64, 1), (128, 1), (64, 5)])
def test_many_jobs_a_processor(cuda, D, T):
    """Jobs of two tiles, of one tile and of few rows follow one another on every processor, many times over."""
    S = 300 // T
    lens = []
    for i in range(S):
        lens += [max(0, (29 * i) % 300 - T + 1 + t) for t in range(T)]
    Case(200, 200, D, 300, lens, T=T, seed=19).check()
    Case(390, 3, D, 130, lens[: 20 * T], T=T, seed=20).check()


@pytest.mark.parametrize("S", [385, 1000])
def test_more_sequences_than_threads(cuda, S):
    """The lengths are summed in several rounds; most sequences are empty or padding, some far between are not."""
    Case(2, 1, 64, 100, [(7 * i) % 130 for i in range(S)], seed=24).check()
    Case(6, 2, 128, 65, [300 if i % 97 == 5 else (0 if i % 2 else -1) for i in range(S)], seed=25, gate=True).check()
    Case(2, 1, 64, 0, [200 if i >= S - 2 else 0 for i in range(S)], seed=26, dtype=torch.float16).check()


def test_same_bits_every_time(cuda):
    c = Case(40, 8, 128, 3000, [5, 900, 64, 65, 1, 0, 2000], seed=14)
    a = c.run().clone()
    for _ in range(5):
        assert torch.equal(c.run(), a)


def test_captured_graph_follows_the_lengths(cuda):
    from volundr_mlx_b200 import ops

    c = Case(10, 2, 128, 600, [400, 300, 129], seed=15)
    lens, P = c.lens.clone(), c.P
    c.run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.run()
    for new, p in (([1, 0, 129], 600), ([400, 300, 0], 64), ([-1, 5, 64], 0), (lens.tolist(), P)):
        c.lens.copy_(torch.tensor(new, dtype=torch.int32))
        c.prefix_len.fill_(p)
        c.P = p
        before = c.out.clone()
        g.replay()
        ops.check_status()
        check_attend(c.out, c.want(), before)


def test_two_graphs_and_two_streams(cuda):
    """Calls that overlap share no scratch: two graphs replayed on two streams give what each gives alone."""
    a, b = Case(40, 8, 128, 4000, [500] * 16, seed=16), Case(40, 8, 128, 5000, [300] * 12, seed=17)
    ra, rb = a.run().clone(), b.run().clone()
    graphs = []
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run()
        c.out.zero_()
        graphs.append((g, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a.out, ra) and torch.equal(b.out, rb)


def test_bad_pages_and_lengths_are_reported(cuda):
    """A page outside the pool reads page 0 instead, a length beyond its page list is cut: both are reported."""
    from volundr_mlx_b200 import ops

    for spoil in ("prefix page", "own page", "prefix length", "own length"):
        c = Case(4, 2, 64, 200, [100, 30], seed=18)
        c.K.nan_to_num_(0, 0, 0)
        c.V.nan_to_num_(0, 0, 0)
        if spoil == "prefix page":
            c.prefix_pages[1] = c.K.shape[0]
        elif spoil == "own page":
            c.table[0, 1] = -1
        elif spoil == "prefix length":
            c.prefix_len.fill_(100000)
        else:
            c.lens[0] = 1 << 30
        c.run()
        with pytest.raises(RuntimeError, match="index outside"):
            ops.check_status()
        assert bool(torch.isfinite(c.out).all())


def test_steps_of_rotate_append_attend(cuda):
    """A batch behind a shared prefix decodes: each step rotates and appends one token per sequence, then attends; every
    step's output against a softmax over the whole history kept in 64 bits."""
    from volundr_mlx_b200 import ops, rotary

    gen = torch.Generator(device="cuda").manual_seed(21)

    def normal(*shape):
        return torch.empty(shape, device="cuda", dtype=torch.bfloat16).normal_(0, 1, generator=gen)

    S, H, KVH, D, P = 5, 10, 2, 128, 150
    freq, m = rotary.frequencies(64, 1e4, scaling="parts", factor=4.0, device="cuda")
    K, V = torch.full((30, KVH, PAGE, D), math.nan, device="cuda", dtype=torch.bfloat16), torch.full((30, KVH, PAGE, D), math.nan, device="cuda", dtype=torch.bfloat16)
    perm = torch.randperm(30, device="cuda", generator=gen).to(torch.int32)
    prefix, table = perm[:3].contiguous(), perm[3:18].view(5, 3).contiguous()
    ar = torch.arange(P, device="cuda", dtype=torch.int32)
    # the prompt goes in once, as one sequence's chunk, through the same append
    ops.kv_append(normal(P, KVH, D), normal(P, KVH, D), K, V, prefix.view(1, 3), ar, freq, seq=torch.zeros_like(ar), magnitude=m)
    plen = torch.tensor([P], device="cuda", dtype=torch.int32)
    slot = torch.tensor([0, 60, 63, -1, 0], device="cuda", dtype=torch.int32)      # sequence 3 is padding
    for b in (1, 2):                                                                # two sequences are already under way
        n = int(slot[b])
        t = torch.arange(n, device="cuda", dtype=torch.int32)
        ops.kv_append(normal(n, KVH, D), normal(n, KVH, D), K, V, table, t + P, freq, slot=t, seq=torch.full_like(t, b), magnitude=m)
    for step in range(8):
        qkv = normal(S, H + 2 * KVH, D)
        q = ops.kv_append(qkv[:, H:H + KVH], qkv[:, H + KVH:], K, V, table, slot + P, freq, slot=slot, q=qkv[:, :H], magnitude=m,
                          q_out=torch.zeros((S, H, D), device="cuda", dtype=torch.bfloat16))
        alone = ops.rope(qkv[:, :H], slot + P, freq, magnitude=m)
        live = slot >= 0
        assert torch.equal(q[live], alone[live])
        lens = torch.where(live, slot + 1, slot)
        out = torch.full_like(q, 7.0)
        before = out.clone()
        ops.attend_prefix(q, K, V, prefix, plen, table, lens, out=out)
        ops.check_status()
        check_attend(out, attend(q, K, V, prefix, P, table, lens, 1), before)
        slot = torch.where(live, slot + 1, slot)


def test_wrappers_refuse(cuda):
    """Wrong shapes, types, strides and gradients never reach a launch."""
    from volundr_mlx_b200 import ops, rotary

    c = Case(4, 2, 64, 100, [30, 40], seed=23)
    a = dict(q=c.q, K=c.K, V=c.V, prefix_pages=c.prefix_pages, prefix_len=c.prefix_len, table=c.table, lens=c.lens)
    ops.attend_prefix(**a)
    wide = torch.zeros((2, 4, 72), device="cuda", dtype=c.q.dtype)
    for bad in (dict(q=c.q.float()), dict(q=c.q.half()), dict(q=c.q[:, :3]), dict(q=wide[:, :, 4:68]), dict(K=c.K.transpose(0, 1)),
                dict(V=c.V[:, :1]), dict(lens=c.lens[:1]), dict(lens=c.lens.long()), dict(prefix_len=c.prefix_len.long()),
                dict(prefix_pages=c.prefix_pages[None]), dict(table=c.table[:1]), dict(table=c.table.cpu()), dict(T=0), dict(T=2),
                dict(scale=0.0), dict(scale=-1.0), dict(gate=c.q[:1]), dict(out=c.q[:, :, :32]),
                dict(q=c.q.clone().requires_grad_(True))):
        with pytest.raises(ValueError):
            ops.attend_prefix(**{**a, **bad})
    freq, _ = rotary.frequencies(64, 1e4, device="cuda")
    pos = torch.zeros(2, device="cuda", dtype=torch.int32)
    k = torch.zeros((2, 2, 64), device="cuda", dtype=c.q.dtype)
    for bad in (dict(pos=pos.long()), dict(freq=freq.float()), dict(freq=torch.ones(33, device="cuda", dtype=torch.float64)),
                dict(out=torch.zeros((2, 2, 32), device="cuda", dtype=c.q.dtype)), dict(x=k.float()), dict(x=k.transpose(1, 2)),
                dict(out=k.transpose(0, 1))):
        with pytest.raises(ValueError):
            ops.rope(**{**dict(x=k, pos=pos, freq=freq), **bad})
    b = dict(k=k, v=k, K=c.K, V=c.V, table=c.table, pos=pos, freq=freq)
    for bad in (dict(v=k[:1]), dict(v=k.half()), dict(K=c.K[:, :1]), dict(table=c.table[0]), dict(slot=pos[:1]), dict(seq=pos.long()),
                dict(q=c.q[:1]), dict(q_out=c.q), dict(table=c.table[:1])):
        with pytest.raises(ValueError):
            ops.kv_append(**{**b, **bad})
    ops.check_status()
