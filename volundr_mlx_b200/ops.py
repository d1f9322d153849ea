"""torch-facing wrappers of the C ABI: tensors in, tensors out, raw pointers and the current stream underneath."""
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
# (These run once per layer and step beside kernels of a few microseconds: every check is one or two attribute reads, and the
# arguments go down as one packed struct.)
PAGE = 64
_TYPES = {BF16: 0, torch.float16: 1}
_raw_stream = torch._C._cuda_getCurrentRawStream      # the stream of torch.cuda.current_stream(index), as an integer


def _refuse(what):
    raise ValueError(what)


def _on(idx, t, name, floating=False):
    """t lives on CUDA device idx and carries no gradient that the operator would lose."""
    if idx < 0:
        _refuse("CUDA tensors are required: there is no CPU path")
    if t.get_device() != idx:
        _refuse(f"{name} is on {t.device}, not on cuda:{idx}")
    if floating and t.requires_grad and torch.is_grad_enabled():
        _refuse(f"{name} requires a gradient: the operator records none")


def _heads(idx, t, name, dtype, rows=None, heads=None, D=None):
    """[rows, heads, D] of `dtype`, the elements of a head side by side, rows and heads strided: its shape and strides."""
    _on(idx, t, name, True)
    sh, st = t.shape, t.stride()
    if t.dtype != dtype or len(sh) != 3:
        _refuse(f"{name}: a [rows, heads, D] tensor of {dtype}")
    if (D is not None and sh[2] != D) or (rows is not None and sh[0] != rows) or (heads is not None and sh[1] != heads):
        _refuse(f"{name}: shape {tuple(sh)}")
    if st[2] != 1 and sh[2] > 1:
        _refuse(f"{name}: the elements of a head must lie side by side")
    return sh, st


def _ints(idx, t, name, *shape):
    _on(idx, t, name)
    if t.dtype != torch.int32 or not t.is_contiguous() or t.shape != shape:
        _refuse(f"{name}: contiguous int32 {shape}")


def _table(idx, t, name):
    _on(idx, t, name)
    if t.dtype != torch.int32 or not t.is_contiguous() or t.dim() != 2:
        _refuse(f"{name}: contiguous int32 [sequences, pages]")
    return t.shape


def _pools(idx, K, V, dtype):
    """K, V: contiguous pages [n_pages, kv heads, PAGE, D]; their shape."""
    _on(idx, K, "K", True)
    _on(idx, V, "V", True)
    sh = K.shape
    if len(sh) != 4 or sh[2] != PAGE or sh != V.shape or K.dtype != dtype or V.dtype != dtype or sh[0] == 0 or sh[1] == 0:
        _refuse(f"K, V: pages [n_pages, kv heads, {PAGE}, D] of {dtype}")
    if not (K.is_contiguous() and V.is_contiguous()):
        _refuse("K, V: contiguous pages")
    return sh


def _turned(idx, freq, D):
    """Rotated elements of a head."""
    if freq is None:
        return 0
    _on(idx, freq, "freq", True)
    n = 2 * freq.numel()
    if freq.dtype != torch.float64 or freq.dim() != 1 or not freq.is_contiguous() or n > D:
        _refuse(f"freq: contiguous float64 [dims / 2], dims at most the head's {D} elements")
    return n


def _launch(idx, fn, what, *args):
    """fn(*args, stream) on the current stream of device idx, that device current."""
    if idx == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(idx))
    else:
        with torch.cuda.device(idx):
            rc = fn(*args, _raw_stream(idx))
    if rc:
        _lib.check(rc, what)


def rope(x, pos, freq, *, interleaved=False, magnitude=1.0, inverse=False, out=None):
    """Rotary positions: the first 2 * len(freq) elements of every head of x [rows, heads, D] turned by pos[row] * freq,
    the rest copied. Pairs are (i, i + len(freq)), or (2i, 2i + 1) when interleaved; the rotated elements are also
    multiplied by `magnitude`. pos int32 [rows]; freq float64 [dims / 2] (rotary.frequencies makes it, scaled for long
    contexts). inverse: the transposed rotation, which is also the gradient of the plain one. out may be x itself (same
    strides); any other overlap with x is the caller's error. The model's own layers rotate inside vk_attn_prep
    (volundr.py:663-664)."""
    idx, dtype = x.get_device(), x.dtype
    if dtype not in _TYPES:
        _refuse("x: bfloat16 or float16")
    (rows, heads, D), xs = _heads(idx, x, "x", dtype)
    _ints(idx, pos, "pos", rows)
    dims = _turned(idx, freq, D)
    if out is None:
        out = torch.empty((rows, heads, D), dtype=dtype, device=x.device)
    os = _heads(idx, out, "out", dtype, rows, heads, D)[1]
    if os != xs and out.data_ptr() == x.data_ptr():
        _refuse("out overlaps x with other strides")
    if rows and heads:
        _launch(idx, _lib.lib().vk_rope, "vk_rope",
                _lib.ROPE_PACK(_TYPES[dtype], rows, heads, D, dims, bool(interleaved), bool(inverse), magnitude, x.data_ptr(), xs[0],
                               xs[1], out.data_ptr(), os[0], os[1], pos.data_ptr(), 0 if freq is None else freq.data_ptr()))
    return out


def kv_append(k, v, K, V, table, pos, freq=None, *, slot=None, seq=None, q=None, q_out=None, interleaved=False, magnitude=1.0):
    """New tokens into the paged cache: row r's keys k[r], rotated by pos[r] (see rope), and values v[r] go to token
    slot[r] (default pos[r]) of sequence seq[r] (default r): page table[seq, slot // 64], row slot % 64 of K, V [n_pages,
    kv heads, 64, D]. With q [rows, heads, D] its rotation lands in q_out, which is returned. A row whose slot is negative
    is padding: nothing of it is written. Rows of one call must name different (seq, slot) places: two rows on one place
    leave a mixture of both. A page outside the pool, or a slot beyond the table, is reported by check_status and
    skipped. slot and pos differ where a sequence's first tokens are a prefix held elsewhere (attend_prefix)."""
    idx, dtype = k.get_device(), k.dtype
    if dtype not in _TYPES:
        _refuse("k: bfloat16 or float16")
    (rows, KVH, D), ks = _heads(idx, k, "k", dtype)
    vs = _heads(idx, v, "v", dtype, rows, KVH, D)[1]
    pages = _pools(idx, K, V, dtype)
    if pages[1] != KVH or pages[3] != D:
        _refuse("K, V: kv heads and head size of k")
    seqs, max_pages = _table(idx, table, "table")
    _ints(idx, pos, "pos", rows)
    if slot is not None:
        _ints(idx, slot, "slot", rows)
    if seq is not None:
        _ints(idx, seq, "seq", rows)
    elif rows > seqs:
        _refuse("more rows than sequences: give seq")
    dims = _turned(idx, freq, D)
    H, qp, qs, op, os = 0, 0, (0, 0), 0, (0, 0)
    if q is not None:
        qsh, qs = _heads(idx, q, "q", dtype, rows, None, D)
        H, qp = qsh[1], q.data_ptr()
        if q_out is None:
            q_out = torch.empty(qsh, dtype=dtype, device=q.device)
        os, op = _heads(idx, q_out, "q_out", dtype, rows, H, D)[1], q_out.data_ptr()
        if os != qs and op == qp:
            _refuse("q_out overlaps q with other strides")
    elif q_out is not None:
        _refuse("q_out without q")
    if rows:
        if not (seqs and max_pages):
            _refuse("table: at least one sequence and one page")
        _launch(idx, _lib.lib().vk_kv_append, "vk_kv_append",
                _lib.APPEND_PACK(_TYPES[dtype], rows, H, KVH, D, dims, bool(interleaved), magnitude, qp, k.data_ptr(), v.data_ptr(),
                                 qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], op, os[0], os[1], K.data_ptr(), V.data_ptr(),
                                 table.data_ptr(), pos.data_ptr(), 0 if slot is None else slot.data_ptr(),
                                 0 if seq is None else seq.data_ptr(), 0 if freq is None else freq.data_ptr(), seqs, max_pages,
                                 pages[0]))
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
    idx, dtype = q.get_device(), q.dtype
    if dtype not in _TYPES:
        _refuse("q: bfloat16 or float16")
    (R, H, D), qs = _heads(idx, q, "q", dtype)
    n_pages, KVH, _, PD = _pools(idx, K, V, dtype)
    if PD != D or D not in (64, 128):
        _refuse("head size: 64 or 128, the same in q and the pages")
    if H == 0 or H % KVH:
        _refuse("query heads: a multiple of the pages' kv heads")
    seqs, max_pages = _table(idx, table, "table")
    if T < 1 or seqs * T != R:
        _refuse("table: one row per T rows of q")
    _ints(idx, lens, "lens", R)
    _ints(idx, prefix_len, "prefix_len", 1)
    _ints(idx, prefix_pages, "prefix_pages", prefix_pages.numel())
    if out is None:
        out = torch.zeros((R, H, D), dtype=dtype, device=q.device)
    os = _heads(idx, out, "out", dtype, R, H, D)[1]
    gp, gs = 0, (0, 0)
    if gate is not None:
        gs, gp = _heads(idx, gate, "gate", dtype, R, H, D)[1], gate.data_ptr()
    qp, op = q.data_ptr(), out.data_ptr()
    if (qp | op | gp) & 15 or (qs[0] | qs[1] | os[0] | os[1] | gs[0] | gs[1]) & 7:
        _refuse("q, out, gate: 16-byte aligned heads")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        _refuse("scale: positive and finite")
    if R:
        L = _lib.lib()
        a = _lib.PREFIX_PACK(_TYPES[dtype], seqs, T, H, KVH, D, scale, qp, qs[0], qs[1], gp, gs[0], gs[1], op, os[0], os[1],
                             K.data_ptr(), V.data_ptr(), n_pages, prefix_pages.data_ptr(), prefix_pages.numel(),
                             prefix_len.data_ptr(), table.data_ptr(), max_pages, lens.data_ptr())
        # scratch of its own per call, from the caching allocator: calls on other streams or in other graphs share nothing
        need = L.vk_attend_prefix_workspace_bytes(a)
        ws = torch.empty(need or 16, dtype=torch.uint8, device=q.device)
        _launch(idx, L.vk_attend_prefix, "vk_attend_prefix", a, ws.data_ptr(), need)
    return out
