"""torch-facing wrappers of the C ABI: tensors in, tensors out, raw pointers and the current stream underneath."""
import ctypes

import torch

from . import _lib

BF16 = torch.bfloat16


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _p(t):
    return None if t is None else t.data_ptr()


class W4Weight:
    """An INT4 affine weight in the GEMM's streaming layout (1152-byte chunks of 32 rows x 64 columns)."""

    def __init__(self, packed, N, K, group):
        self.packed, self.N, self.K, self.group = packed, N, K, group

    @property
    def nbytes(self):
        return self.packed.numel()


def w4_repack(w, scales, biases, group=64) -> W4Weight:
    """Reference layout (uint32 [N, K/8] codes as int32 tensor, bf16 scales/biases [N, K/group]) -> W4Weight."""
    L = _lib.lib()
    N, K = w.shape[0], w.shape[1] * 8
    assert w.dtype == torch.int32 and scales.dtype == BF16 and biases.dtype == BF16
    assert scales.shape == (N, K // group) == biases.shape
    packed = torch.empty(L.vk_w4_packed_bytes(N, K), dtype=torch.uint8, device=w.device)
    _lib.check(L.vk_w4_repack(_p(w.contiguous()), _p(scales.contiguous()), _p(biases.contiguous()), N, K, group,
                              _p(packed), _stream()), "vk_w4_repack")
    return W4Weight(packed, N, K, group)


def w4_dequant(w, scales, biases, group=64):
    L = _lib.lib()
    N, K = w.shape[0], w.shape[1] * 8
    out = torch.empty((N, K), dtype=BF16, device=w.device)
    _lib.check(L.vk_w4_dequant(_p(w.contiguous()), _p(scales.contiguous()), _p(biases.contiguous()), N, K, group,
                               _p(out), _stream()), "vk_w4_dequant")
    return out


_ws = {}


def workspace(nbytes, device):
    """One grow-only scratch buffer per device: split-K arrival counters (zero between launches) then the partial
    sums. Allocated outside the step's hot loop."""
    key = str(device)
    buf = _ws.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.zeros(max(nbytes, 1 << 25), dtype=torch.uint8, device=device)
        _ws[key] = buf
    return buf


_tile_ws = {}


def tile_workspace(nbytes, device):
    """Scratch of vk_w4_gemm_tile (arrival counters, zero between launches, activation tiles, partial sums): a buffer of
    its own, since the tile kernel's activation tiles would otherwise land on the streaming kernel's counters."""
    key = str(device)
    buf = _tile_ws.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.zeros(max(nbytes, 1 << 25), dtype=torch.uint8, device=device)
        _tile_ws[key] = buf
    return buf


def w4_gemm(x, wt: W4Weight, out=None):
    """y[M, N] = x[M, K] . dequant(W)^T, bf16 in / out, fp32 accumulation."""
    L = _lib.lib()
    assert x.dtype == BF16 and x.dim() == 2 and x.shape[1] == wt.K and x.stride(1) == 1
    M = x.shape[0]
    if out is None:
        out = torch.empty((M, wt.N), dtype=BF16, device=x.device)
    need = L.vk_w4_workspace_bytes(M, wt.N, wt.K)
    ws = workspace(need, x.device)
    _lib.check(L.vk_w4_gemm(_p(wt.packed), _p(x), x.stride(0), _p(out), out.stride(0), M, wt.N, wt.K, _p(ws),
                            ws.numel(), _stream()), "vk_w4_gemm")
    return out


def w4_gemm_tile(x, wt: W4Weight, out=None):
    """The same product on the tcgen05 tensor cores (tiles of 128 rows): meant for M >= 64."""
    L = _lib.lib()
    assert x.dtype == BF16 and x.dim() == 2 and x.shape[1] == wt.K and x.stride(1) == 1
    M = x.shape[0]
    if out is None:
        out = torch.empty((M, wt.N), dtype=BF16, device=x.device)
    ws = tile_workspace(L.vk_w4_tile_workspace_bytes_n(M, wt.N, wt.K), x.device)
    _lib.check(L.vk_w4_gemm_tile(_p(wt.packed), _p(x), x.stride(0), _p(out), out.stride(0), M, wt.N, wt.K, _p(ws),
                                 ws.numel(), _stream()), "vk_w4_gemm_tile")
    return out


class BF16Weight:
    """A bf16 weight [N, K] in the streaming kernel's fragment order (4096-byte chunks of 32 rows x 64 columns)."""

    def __init__(self, packed, N, K):
        self.packed, self.N, self.K = packed, N, K

    @property
    def nbytes(self):
        return self.packed.numel()


def bf16_repack(W) -> BF16Weight:
    L = _lib.lib()
    N, K = W.shape
    assert W.dtype == BF16 and W.is_contiguous()
    packed = torch.empty(L.vk_bf16_packed_bytes(N, K), dtype=torch.uint8, device=W.device)
    _lib.check(L.vk_bf16_repack(_p(W), N, K, _p(packed), _stream()), "vk_bf16_repack")
    return BF16Weight(packed, N, K)


def bf16_gemm(x, wt: BF16Weight, out=None):
    """y[M, N] = x[M, K] . W^T for a repacked bf16 weight."""
    L = _lib.lib()
    assert x.dtype == BF16 and x.dim() == 2 and x.shape[1] == wt.K and x.stride(1) == 1
    M = x.shape[0]
    if out is None:
        out = torch.empty((M, wt.N), dtype=BF16, device=x.device)
    ws = workspace(L.vk_bf16_workspace_bytes(min(M, 16), wt.N, wt.K), x.device)
    _lib.check(L.vk_bf16_gemm_packed(_p(wt.packed), _p(x), x.stride(0), _p(out), out.stride(0), M, wt.N, wt.K, _p(ws),
                                     ws.numel(), _stream()), "vk_bf16_gemm_packed")
    return out


_status_buf = {}


def check_status(device=None):
    """Read and clear the device status word (synchronises); raises if a kernel recorded an error."""
    L = _lib.lib()
    device = device or torch.device("cuda", torch.cuda.current_device())
    key = str(device)
    if key not in _status_buf:
        _status_buf[key] = torch.zeros(1, dtype=torch.int32, device=device)
    buf = _status_buf[key]
    _lib.check(L.vk_status_fetch(_p(buf), _stream()), "vk_status_fetch")
    code = int(buf.item())
    if code:
        # a wait that ran out may have left a split-K arrival counter behind: put the scratch buffers' heads back to zero
        for pool in (_ws, _tile_ws):
            if key in pool:
                pool[key][: 1 << 14].zero_()
        raise RuntimeError("volundr_b200 device status: " + L.vk_status_string(code).decode())


# ---------------------------------------------------------------- rotary positions, paged append, shared-prefix attention
PAGE = 64
_TYPES = {BF16: 0, torch.float16: 1}


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _same(dev, **tensors):
    """Every given tensor lives on the CUDA device `dev` and carries no gradient these operators would lose."""
    _need(dev.type == "cuda", "CUDA tensors are required: there is no CPU path")
    for name, t in tensors.items():
        if t is not None:
            _need(t.device == dev, f"{name} is on {t.device}, not on {dev}")
            _need(not (t.requires_grad and torch.is_grad_enabled()), f"{name} requires a gradient: the operator records none")


def _heads(name, t, dtype, rows=None, heads=None, D=None):
    """[rows, heads, D] of a 16-bit type, elements of a head side by side; rows and heads may be strided."""
    _need(t.dim() == 3 and t.dtype == dtype, f"{name}: a [rows, heads, D] tensor of {dtype}")
    _need(all(w is None or n == w for n, w in zip(t.shape, (rows, heads, D))), f"{name}: shape {tuple(t.shape)}")
    _need(t.shape[2] <= 1 or t.stride(2) == 1, f"{name}: the elements of a head must lie side by side")


def _ints(name, t, *shape):
    _need(t.dtype == torch.int32 and t.is_contiguous() and tuple(t.shape) == shape, f"{name}: contiguous int32 {shape}")


def _pool(K, V, dtype):
    for name, t in (("K", K), ("V", V)):
        _need(t.dim() == 4 and t.dtype == dtype and t.is_contiguous() and t.shape == K.shape and t.shape[2] == PAGE,
              f"{name}: contiguous pages [n_pages, kv heads, {PAGE}, D] of {dtype}")


def _turns(freq, D, dev):
    if freq is None:
        return 0
    _same(dev, freq=freq)
    _need(freq.dtype == torch.float64 and freq.dim() == 1 and freq.is_contiguous(), "freq: contiguous float64 [dims / 2]")
    _need(2 * freq.numel() <= D, f"freq: {2 * freq.numel()} rotated elements in a head of {D}")
    return 2 * freq.numel()


class _On:
    """The launch's device made current (only when it is not), so that the stream and the launch belong to the tensors."""

    def __init__(self, dev):
        self.guard = None if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return _stream()

    def __exit__(self, *e):
        if self.guard is not None:
            self.guard.__exit__(*e)


def rope(x, pos, freq, *, interleaved=False, magnitude=1.0, inverse=False, out=None):
    """Rotary positions: the first 2 * len(freq) elements of every head of x [rows, heads, D] turned by pos[row] * freq,
    the rest copied. Pairs are (i, i + len(freq)), or (2i, 2i + 1) when interleaved; the rotated elements are also
    multiplied by `magnitude`. pos int32 [rows]; freq float64 [dims / 2] (rotary.frequencies makes it, scaled for long
    contexts). inverse: the transposed rotation, which is also the gradient of the plain one. out may be x itself (same
    strides); any other overlap with x is the caller's error. The model's own layers rotate inside vk_attn_prep
    (volundr.py:663-664)."""
    _same(x.device, pos=pos, x=x, out=out)
    _need(x.dtype in _TYPES, "x: bfloat16 or float16")
    _heads("x", x, x.dtype)
    rows, heads, D = x.shape
    _ints("pos", pos, rows)
    dims = _turns(freq, D, x.device)
    if out is None:
        out = torch.empty((rows, heads, D), dtype=x.dtype, device=x.device)
    _heads("out", out, x.dtype, rows, heads, D)
    _need(out.data_ptr() != x.data_ptr() or out.stride() == x.stride(), "out overlaps x with other strides")
    if rows == 0 or heads == 0:
        return out
    with _On(x.device) as st:
        _lib.check(_lib.lib().vk_rope(_TYPES[x.dtype], _p(x), x.stride(0), x.stride(1), _p(out), out.stride(0), out.stride(1),
                                      _p(pos), _p(freq), dims, int(interleaved), int(inverse), float(magnitude), rows, heads, D,
                                      st), "vk_rope")
    return out


def kv_append(k, v, K, V, table, pos, freq=None, *, slot=None, seq=None, q=None, q_out=None, interleaved=False, magnitude=1.0):
    """New tokens into the paged cache: row r's keys k[r], rotated by pos[r] (see rope), and values v[r] go to token
    slot[r] (default pos[r]) of sequence seq[r] (default r): page table[seq, slot // 64], row slot % 64 of K, V [n_pages,
    kv heads, 64, D]. With q [rows, heads, D] its rotation lands in q_out, which is returned. A row whose slot is negative
    is padding: nothing of it is written. Rows of one call must name different (seq, slot) places: two rows on one place
    leave a mixture of both. A page outside the pool, or a slot beyond the table, is reported by check_status and
    skipped. slot and pos differ where a sequence's first tokens are a prefix held elsewhere (attend_prefix)."""
    dev = k.device
    _same(dev, k=k, v=v, K=K, V=V, table=table, pos=pos, slot=slot, seq=seq, q=q, q_out=q_out)
    _need(k.dtype in _TYPES, "k: bfloat16 or float16")
    _heads("k", k, k.dtype)
    rows, KVH, D = k.shape
    _heads("v", v, k.dtype, rows, KVH, D)
    _pool(K, V, k.dtype)
    _need(K.shape[0] > 0 and K.shape[1] == KVH and K.shape[3] == D, "K, V: kv heads and head size of k")
    _need(table.dim() == 2 and table.numel() > 0, "table: [sequences, pages]")
    _ints("table", table, *table.shape)
    for name, t in (("pos", pos), ("slot", slot), ("seq", seq)):
        if t is not None:
            _ints(name, t, rows)
    _need(seq is not None or rows <= table.shape[0], "more rows than sequences: give seq")
    a = _lib.AppendArgs()
    a.dims = _turns(freq, D, dev)
    if q is not None:
        _heads("q", q, k.dtype, rows, None, D)
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        _heads("q_out", q_out, k.dtype, *q.shape)
        _need(q_out.data_ptr() != q.data_ptr() or q_out.stride() == q.stride(), "q_out overlaps q with other strides")
        a.Hq, a.q, a.q_row, a.q_head = q.shape[1], _p(q), q.stride(0), q.stride(1)
        a.q_out, a.qo_row, a.qo_head = _p(q_out), q_out.stride(0), q_out.stride(1)
    else:
        _need(q_out is None, "q_out without q")
    if rows == 0:
        return q_out
    a.dtype, a.rows, a.KVH, a.D, a.interleaved, a.magnitude = _TYPES[k.dtype], rows, KVH, D, int(interleaved), float(magnitude)
    a.k, a.v, a.k_row, a.k_head, a.v_row, a.v_head = _p(k), _p(v), k.stride(0), k.stride(1), v.stride(0), v.stride(1)
    a.K, a.V, a.table, a.pos, a.slot, a.seq, a.freq = _p(K), _p(V), _p(table), _p(pos), _p(slot), _p(seq), _p(freq)
    a.n_seqs, a.max_pages, a.n_pages = table.shape[0], table.shape[1], K.shape[0]
    with _On(dev) as st:
        _lib.check(_lib.lib().vk_kv_append(ctypes.byref(a), st), "vk_kv_append")
    return q_out


def attend_prefix(q, K, V, prefix_pages, prefix_len, table, lens, *, T=1, scale=None, gate=None, out=None):
    """Decode attention of sequences that share a prompt prefix: row r = b * T + t of q [B * T, heads, D] (the T newest
    tokens of B sequences; D 64 or 128) attends the first prefix_len[0] tokens of the pages prefix_pages [n] and the first
    lens[r] tokens of its sequence's own pages table[b], all in the pool K, V [n_pages, kv heads, 64, D]:
    softmax(scale q k) v, scale 1 / sqrt(D) by default, times sigmoid(gate) when a gate [B * T, heads, D] is given. The
    prefix is read once for the whole batch. A row with lens < 0 is padding: its output stays as it was. A row that
    sees no key at all gets zeros. prefix_len and lens are int32 on the device, so that a captured graph follows them.
    Keys and values behind a sequence's last visible token may hold anything; those that one of a sequence's T rows sees
    must be finite for all of its rows. Sums and statistics are fp32, probabilities meet the values in the
    storage type. The per-sequence form without a shared part is vk_attend_decode."""
    dev = q.device
    _same(dev, q=q, K=K, V=V, prefix_pages=prefix_pages, prefix_len=prefix_len, table=table, lens=lens, gate=gate, out=out)
    _need(q.dtype in _TYPES, "q: bfloat16 or float16")
    _heads("q", q, q.dtype)
    R, H, D = q.shape
    _pool(K, V, q.dtype)
    KVH = K.shape[1]
    _need(D in (64, 128) and K.shape[3] == D, "head size: 64 or 128, the same in q and the pages")
    _need(K.shape[0] > 0 and KVH > 0 and H > 0 and H % KVH == 0, "query heads: a multiple of the pages' kv heads")
    _need(T >= 1 and R % T == 0 and table.dim() == 2 and table.shape[0] == R // T, "table: one row per T rows of q")
    _ints("table", table, *table.shape)
    _ints("lens", lens, R)
    _ints("prefix_len", prefix_len, 1)
    _need(prefix_pages.dim() == 1, "prefix_pages: [n]")
    _ints("prefix_pages", prefix_pages, *prefix_pages.shape)
    if out is None:
        out = torch.zeros((R, H, D), dtype=q.dtype, device=dev)
    for name, t in (("q", q), ("gate", gate), ("out", out)):
        if t is not None:
            _heads(name, t, q.dtype, R, H, D)
            _need(t.data_ptr() % 16 == 0 and t.stride(0) % 8 == 0 and t.stride(1) % 8 == 0, f"{name}: 16-byte aligned heads")
    scale = D ** -0.5 if scale is None else float(scale)
    _need(0.0 < scale < float("inf"), "scale: positive and finite")
    if R == 0:
        return out
    a = _lib.PrefixArgs()
    a.dtype, a.seqs, a.T, a.Hq, a.KVH, a.D, a.scale = _TYPES[q.dtype], R // T, T, H, KVH, D, scale
    a.q, a.q_row, a.q_head = _p(q), q.stride(0), q.stride(1)
    if gate is not None:
        a.gate, a.gate_row, a.gate_head = _p(gate), gate.stride(0), gate.stride(1)
    a.out, a.out_row, a.out_head = _p(out), out.stride(0), out.stride(1)
    a.K, a.V, a.n_pages = _p(K), _p(V), K.shape[0]
    a.prefix_pages, a.max_prefix_pages, a.prefix_len = _p(prefix_pages), prefix_pages.numel(), _p(prefix_len)
    a.table, a.max_pages, a.lens = _p(table), table.shape[1], _p(lens)
    L = _lib.lib()
    with _On(dev) as st:
        # scratch of its own per call, from the caching allocator: calls on other streams or in other graphs share nothing
        need = L.vk_attend_prefix_workspace_bytes(ctypes.byref(a))
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        _lib.check(L.vk_attend_prefix(ctypes.byref(a), _p(ws), ws.numel(), st), "vk_attend_prefix")
    return out
