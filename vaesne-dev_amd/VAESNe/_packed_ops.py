"""Autograd operators of the packed-sequence layers (VAESNe.PackedLayers), each backed by
libvaesne_hip.so: attention over packed sequences with an optional relative position bias, the
gated norm join, activations kept in 8 bits (include/vaesne_hip.h).

Tensors are fp32, bf16 or fp16, all of one call the same; sums and statistics are fp32.  Launches
go to the current stream of the tensors' device.  Nothing synchronises, except a plan's tables,
which are copied to the device when a shape of call first needs them.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _capture, _defer, _lib
from ._lib import lib
from ._ops import _rows

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
KINDS = {"rms": 0, "layer": 1}
MAX_TOKENS = (1 << 30) - 64                               # (csrc/packed_attention.hip's)


def _fields(spec):
    out = []
    for kind, names in spec:
        out += [(n, kind) for n in names.split()]
    return out


class _AttnArgs(C.Structure):
    """vaesne_packed_attn"""
    _fields_ = _fields([
        (C.c_int, "type Hq Hkv D causal num_buckets max_distance nseq"), (C.c_float, "scale"),
        (C.c_int, "max_q max_k q_tile k_tile n_q_tiles n_k_tiles"), (C.c_int64, "total_q total_k"),
        (C.c_void_p, "q_tiles k_tiles q k v"),
        (C.c_int64, "q_ts q_hs k_ts k_hs v_ts v_hs"), (C.c_void_p, "o lse table lut dout"),
        (C.c_int64, "do_ts do_hs"), (C.c_void_p, "dq dk dv dtable workspace")])


class _NormArgs(C.Structure):
    """vaesne_gated_norm"""
    _fields_ = _fields([
        (C.c_int, "type kind gate_kind C"), (C.c_int64, "rows"), (C.c_float, "residual_scale eps"),
        (C.c_void_p, "x branch gate pre_w pre_b post_w post_b"), (C.c_int64, "ldx ldbranch ldgate"),
        (C.c_void_p, "y n stats dy dn"), (C.c_int64, "lddy lddn"),
        (C.c_void_p, "dx dbranch dgate dpre_w dpre_b dpost_w dpost_b workspace")])


_FN = {}


def _lib_call(name, device, *args):
    """vaesne_<name>(*args, stream) on `device`'s current stream, with `device` current; raises on a HIP
    error as _lib.lib does.  (Looked up once, and the raw stream asked for: these calls last a few
    microseconds on the device.)"""
    fn = _FN.get(name)
    if fn is None:
        fn = _FN[name] = getattr(_lib.load(), "vaesne_" + name)
    index = device.index
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        raise RuntimeError(f"vaesne_{name} failed: hipError {rc}")


def _type_of(name, *ts):
    """The C type of tensors that must share one type and one ROCm device (and carry no tangent: where no
    gradient is asked for the autograd function is passed by, and would lose it)."""
    if forward_ad._current_level >= 0:
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{name}: there is no forward-mode derivative")
    _lib.require_device(*ts)
    first = ts[0]
    if first.dtype not in TYPES:
        raise TypeError(f"{name}: tensors are float32, bfloat16 or float16, not {first.dtype}")
    for t in ts:
        if t is not None and t.dtype != first.dtype:
            raise TypeError(f"{name}: every tensor has one type, got {first.dtype} and {t.dtype}")
        if t is not None and t.device != first.device:
            raise RuntimeError(f"{name}: every tensor is on one device, got {first.device} and {t.device}")
    return TYPES[first.dtype]


def _ws(nbytes, device):
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=device)


# ---------------------------------------------------------------------------
# attention over packed sequences
# ---------------------------------------------------------------------------
def _lengths(lengths, name):
    if isinstance(lengths, torch.Tensor):
        if lengths.is_floating_point() or lengths.dim() != 1:
            raise ValueError(f"PackedSequences: {name} is a list of whole numbers")
        lengths = lengths.tolist()
    out = [int(n) for n in lengths]
    if any(n < 0 or n != m for n, m in zip(out, lengths)):
        raise ValueError(f"PackedSequences: {name} are whole numbers from 0 up")
    if sum(out) > MAX_TOKENS:
        raise ValueError(f"PackedSequences: {name} add up to more than 2^30 - 64 tokens")
    return out


def tile_table(nq, nk, side, tile, causal):
    """[n][8] rows {first query token, first key token, queries, keys, first position} of every tile of
    `tile` queries ("q") or keys ("k"), most work first: the keys its last query sees, or the queries that
    see its first key."""
    n = nq if side == "q" else nk
    count = -(-n // tile)
    seq = np.repeat(np.arange(len(n)), count)
    first = (np.arange(len(seq)) - np.repeat(np.cumsum(count) - count, count)) * tile
    q, k = nq[seq], nk[seq]
    if side == "q":
        work = np.clip(first + tile + k - q, 0, k) if causal else k
    else:
        work = np.clip(k - first, 0, q) if causal else q
    order = np.argsort(-work, kind="stable")
    out = np.zeros((len(seq), 8), dtype=np.int32)
    out[:, :5] = np.stack([(np.cumsum(nq) - nq)[seq], (np.cumsum(nk) - nk)[seq], q, k, first], 1)[order]
    return out


class PackedSequences:
    """Where the sequences of a packed batch lie: `lengths` queries and `key_lengths` keys (default:
    the same) of each, one behind the other.  A sequence's queries are the LAST ones of its keys'
    positions: one new token over a cache of n keys is lengths 1, key_lengths n.

    Make it once per batch, on the host, and share it between layers; the first call that needs a table
    copies it to the device and waits for the stream.  It keeps device tables, so a captured graph that used it needs it alive; use it once before capturing,
    since a table that is still missing cannot be copied to the device inside a capture.
    training_step never captures a step that uses one: a replay would keep its first batch's lengths."""

    def __init__(self, lengths, key_lengths=None, device="cuda"):
        self.lengths = _lengths(lengths, "lengths")
        self.key_lengths = self.lengths if key_lengths is None else _lengths(key_lengths, "key_lengths")
        if len(self.lengths) != len(self.key_lengths):
            raise ValueError("PackedSequences: as many lengths as key_lengths")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError("VAESNe (MI355X build) runs on ROCm devices only: PackedSequences needs a 'cuda' (HIP) "
                               "device; there is no CPU path.")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._q = np.asarray(self.lengths, dtype=np.int64)
        self._k = np.asarray(self.key_lengths, dtype=np.int64)
        self.total, self.total_keys = int(self._q.sum()), int(self._k.sum())
        self.longest = max(self.lengths, default=0)
        self.longest_keys = max(self.key_lengths, default=0)
        self._tables = {}
        self._calls = {}
        self._index = None

    def __getstate__(self):
        # a copy makes its own tables: the kept calls hold the addresses of this one's
        return {**self.__dict__, "_tables": {}, "_calls": {}}

    @classmethod
    def from_mask(cls, mask):
        """The sequences of a padded batch: `mask` [B, L] on a ROCm device, True = ignore (as
        key_padding_mask).  Reads the mask once (a synchronisation).  `pack` and `unpack` of the
        result go between the padded and the packed form."""
        _lib.require_device(mask)
        if mask.dim() != 2:
            raise ValueError("PackedSequences.from_mask: mask is [B, L]")
        keep = mask == 0 if mask.dtype != torch.bool else ~mask
        at = torch.nonzero(keep.reshape(-1)).reshape(-1)
        out = cls(keep.sum(1).tolist(), device=mask.device)  # (waits for `at` too: any stream may read it)
        out._index = (at, tuple(mask.shape))
        return out

    def _indexes(self, name):
        """from_mask's places and shape; the places are noted on the stream that will read them."""
        if self._index is None:
            raise RuntimeError(f"PackedSequences.{name}: only for sequences made by from_mask")
        _capture.refuse_in_step("PackedSequences")
        self._index[0].record_stream(torch.cuda.current_stream(self.device))
        return self._index

    def pack(self, x):
        """Padded [B, L, ...] -> packed [total, ...] (from_mask's sequences)."""
        at, shape = self._indexes("pack")
        if tuple(x.shape[:2]) != shape:
            raise ValueError(f"PackedSequences.pack: x is {tuple(x.shape)}, the mask was {shape}")
        return x.reshape(shape[0] * shape[1], *x.shape[2:]).index_select(0, at)

    def unpack(self, x):
        """Packed [total, ...] -> padded [B, L, ...], zeros in the masked places."""
        at, shape = self._indexes("unpack")
        if x.shape[0] != self.total:
            raise ValueError(f"PackedSequences.unpack: x has {x.shape[0]} rows, the sequences {self.total}")
        out = x.new_zeros((shape[0] * shape[1], *x.shape[1:])).index_copy(0, at, x)
        return out.reshape(*shape, *x.shape[1:])

    def _upload(self, array):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("PackedSequences: a table is still missing and cannot be made inside a graph capture; "
                               "run the same call once before capturing")
        return torch.from_numpy(array).to(self.device)       # (waits for the copy: any stream may read it)

    def _table(self, side, tile, causal):
        """tile_table's rows on the device, how many, and the stream whose memory they are in."""
        key = (side, tile, bool(causal))
        got = self._tables.get(key)
        if got is None:
            table = tile_table(self._q, self._k, side, tile, causal)
            got = self._tables[key] = (self._upload(table.reshape(-1)) if len(table) else None, len(table),
                                       torch._C._cuda_getCurrentRawStream(self.device.index))
        return got

    def _call(self, type_, Hq, Hkv, D, causal, buckets, backward):
        """One shape of call: the struct's plan fields, the workspace bytes, the device tables."""
        key = (type_, Hq, Hkv, D, causal, buckets and (buckets.num_buckets, buckets.max_distance), backward)
        got = self._calls.get(key)
        if got is None:
            a = _AttnArgs(type=type_, Hq=Hq, Hkv=Hkv, D=D, causal=int(causal), nseq=len(self.lengths), scale=1.0,
                          max_q=self.longest, max_k=self.longest_keys, total_q=self.total, total_k=self.total_keys)
            if buckets is not None:
                a.num_buckets, a.max_distance = buckets.num_buckets, buckets.max_distance
                a.table = a.dtable = 16                      # (any address: sizes only)
            qt, kt = C.c_int(), C.c_int()
            lib.packed_attn_tiles(C.addressof(a), int(backward), C.byref(qt), C.byref(kt))
            a.q_tile, a.k_tile = qt.value, kt.value
            tables = [self._table("q", a.q_tile, causal)]
            a.q_tiles, a.n_q_tiles = None if tables[0][0] is None else tables[0][0].data_ptr(), tables[0][1]
            if backward:
                tables.append(self._table("k", a.k_tile, causal))
                a.k_tiles, a.n_k_tiles = None if tables[1][0] is None else tables[1][0].data_ptr(), tables[1][1]
            ws = lib.packed_attn_workspace(C.addressof(a), int(backward))
            if ws < 0:
                raise RuntimeError("packed_attention: sizes out of range")
            a.table = a.dtable = None
            got = self._calls[key] = (bytes(a), ws, [(t, s) for t, _, s in tables if t is not None])
        return got

    def _args(self, call):
        """A fresh argument struct of `call`; the tables are noted on the stream that will read them."""
        _capture.refuse_in_step("PackedSequences")
        raw = torch._C._cuda_getCurrentRawStream(self.device.index)
        for t, stream in call[2]:
            if stream != raw:
                t.record_stream(torch.cuda.current_stream(self.device))
        return _AttnArgs.from_buffer_copy(call[0])


class RelativeBuckets:
    """Buckets of the relative position (key position minus query position) for a learned bias.

    Half of the buckets (of each direction's share, when bidirectional) hold one distance each; the
    rest grow with the distance's logarithm up to `max_distance`, beyond which all share the last.
    Unidirectional buckets put every key behind the query into bucket 0.  Borders are found
    in whole numbers, so no rounding moves a distance across one."""

    def __init__(self, num_buckets=32, max_distance=128, bidirectional=True):
        num_buckets, max_distance = int(num_buckets), int(max_distance)
        m = num_buckets // 2 if bidirectional else num_buckets
        near = m // 2
        if num_buckets < 2 or (bidirectional and num_buckets % 2) or near < 1:
            raise ValueError("RelativeBuckets: at least 2 buckets in each direction (an even number when bidirectional)")
        if num_buckets > 1024:
            raise ValueError("RelativeBuckets: at most 1024 buckets")
        if not near < max_distance <= 512:
            raise ValueError(f"RelativeBuckets: max_distance lies above {near} (the exact distances) and is at most 512")
        self.num_buckets, self.max_distance, self.bidirectional = num_buckets, max_distance, bool(bidirectional)
        wide = m - near
        # distance n >= near lies in bucket near + k: the largest k < wide with n^wide >= near^(wide-k) max^k
        border = [near ** (wide - k) * max_distance ** k for k in range(wide)]
        of, k = [], 0
        for n in range(max_distance + 1):
            if n < near:
                of.append(n)
                continue
            power = n ** wide
            while k + 1 < wide and power >= border[k + 1]:
                k += 1
            of.append(near + k)
        behind = [m + b for b in of[1:]] if bidirectional else [0] * max_distance
        self.lut = torch.tensor(of[:0:-1] + [of[0]] + behind, dtype=torch.int32)     # positions -R .. R
        self._dev = {}

    def on(self, device):
        """The table [2 max_distance + 1] of buckets on `device` (copied there once)."""
        got = self._dev.get(device)
        if got is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("RelativeBuckets: the bucket table is not on the device yet and cannot be copied "
                                   "inside a graph capture; run the same call once before capturing")
            got = self._dev[device] = (self.lut.to(device), torch._C._cuda_getCurrentRawStream(device.index))
        if torch._C._cuda_getCurrentRawStream(device.index) != got[1]:
            got[0].record_stream(torch.cuda.current_stream(device))
        return got[0]

    def __getstate__(self):
        return {**self.__dict__, "_dev": {}}


def _head_rows(t):
    """t [T, H, D] with unit-stride, 16-byte aligned rows (a copy where it has none)."""
    n = t.element_size()
    s = t.stride()
    if s[2] == 1 and s[0] * n % 16 == 0 and s[1] * n % 16 == 0 and t.data_ptr() % 16 == 0 and max(s) < 1 << 21:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _attn_fwd(q, k, v, seqs, call, scale, table, lut):
    a = seqs._args(call)
    a.scale = scale
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    ws = _ws(call[1], q.device)
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_ts, a.q_hs, _ = q.stride()
    a.k_ts, a.k_hs, _ = k.stride()
    a.v_ts, a.v_hs, _ = v.stride()
    a.o, a.lse, a.workspace = o.data_ptr(), lse.data_ptr(), ws.data_ptr()
    if table is not None:
        a.table, a.lut = table.data_ptr(), lut.data_ptr()
    _lib_call("packed_attn_fwd", q.device, C.addressof(a))
    return o, lse


class PackedAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, seqs, call, back, scale, lut):
        _defer.count_uses(*([] if table is None else [table]))
        tab = None if table is None else table.contiguous()
        o, lse = _attn_fwd(q, k, v, seqs, call, scale, tab, lut)
        ctx.seqs, ctx.back, ctx.scale, ctx.lut = seqs, back, scale, lut
        ctx.save_for_backward(q, k, v, o, lse, tab)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, table = ctx.saved_tensors
        do = _head_rows(do)
        a = ctx.seqs._args(ctx.back)
        a.scale = ctx.scale
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        ws = _ws(ctx.back[1], q.device)
        a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
        a.q_ts, a.q_hs, _ = q.stride()
        a.k_ts, a.k_hs, _ = k.stride()
        a.v_ts, a.v_hs, _ = v.stride()
        a.o, a.lse, a.dout, a.workspace = o.data_ptr(), lse.data_ptr(), do.data_ptr(), ws.data_ptr()
        a.do_ts, a.do_hs, _ = do.stride()
        a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        dtable = None
        if table is not None:
            a.table, a.lut = table.data_ptr(), ctx.lut.data_ptr()
            if ctx.needs_input_grad[3]:
                dtable = torch.empty_like(table)
                a.dtable = dtable.data_ptr()
        _lib_call("packed_attn_bwd", q.device, C.addressof(a))
        ng = ctx.needs_input_grad
        return dq if ng[0] else None, dk if ng[1] else None, dv if ng[2] else None, dtable, None, None, None, None, None


def packed_attention(q, k, v, seqs, causal=False, scale=None, bias=None, buckets=None):
    """Softmax attention over packed sequences (PackedLayers.packed_attention)."""
    type_ = _type_of("packed_attention", q, k, v, bias)
    if not isinstance(seqs, PackedSequences):
        raise TypeError("packed_attention: seqs is a PackedSequences")
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or q.shape[2] != k.shape[2]:
        raise ValueError("packed_attention: q is [queries, heads, dim], k and v are [keys, key heads, dim]")
    Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[:2]
    if q.device != seqs.device:
        raise RuntimeError(f"packed_attention: the tensors are on {q.device}, the sequences on {seqs.device}")
    if Tq != seqs.total or Tk != seqs.total_keys:
        raise ValueError(f"packed_attention: {Tq} queries and {Tk} keys, the sequences hold {seqs.total} and "
                         f"{seqs.total_keys}")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"packed_attention: head dim is a multiple of 8 up to 128, not {D}")
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise ValueError(f"packed_attention: {Hq} heads do not share {Hkv} key heads evenly")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("packed_attention: scale is a positive number")
    if (bias is None) != (buckets is None):
        raise ValueError("packed_attention: bias and buckets go together")
    lut = None
    if bias is not None:
        if not isinstance(buckets, RelativeBuckets):
            raise TypeError("packed_attention: buckets is a RelativeBuckets")
        if tuple(bias.shape) != (buckets.num_buckets, Hq):
            raise ValueError(f"packed_attention: bias is [buckets, heads] = {(buckets.num_buckets, Hq)}, not "
                             f"{tuple(bias.shape)}")
        lut = buckets.on(q.device)
    q, k, v = _head_rows(q), _head_rows(k), _head_rows(v)
    causal = bool(causal)
    call = seqs._call(type_, Hq, Hkv, D, causal, buckets, False)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                    (bias is not None and bias.requires_grad)):
        back = seqs._call(type_, Hq, Hkv, D, causal, buckets, True)
        return PackedAttnFn.apply(q, k, v, bias, seqs, call, back, scale, lut)
    return _attn_fwd(q, k, v, seqs, call, scale, None if bias is None else bias.contiguous(), lut)[0]


# ---------------------------------------------------------------------------
# gated norm join
# ---------------------------------------------------------------------------
def _norm_args(x, branch, pre_w, post_w, pre_b, post_b, gate, scale, kind, eps, type_):
    """(struct, tensors it points to, rows): inputs with uniform rows, parameters contiguous."""
    width = x.shape[-1]
    xr, rows, ldx = _rows(x)
    br, _, ldb = (None, 0, 0) if branch is None else _rows(branch)
    gk, gr, ldg = 0, None, 0
    if gate is not None:
        if gate.dim() == 1 and x.dim() != 1:
            gk, gr = 1, gate.contiguous()
        else:
            gk = 2
            gr, _, ldg = _rows(gate)
    params = [None if t is None else t.contiguous() for t in (pre_w, pre_b, post_w, post_b)]
    p = [None if t is None else t.data_ptr() for t in (xr, br, gr, *params)]
    a = _NormArgs(type_, kind, gk, width, rows, scale, eps, *p, ldx, ldb, ldg)
    return a, (xr, br, gr, *params), rows


def _norm_fwd(a, x, branch, rows, want_stats):
    n = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if branch is not None else None
    stats = torch.empty((rows, 4), dtype=torch.float32, device=x.device) if want_stats else None
    a.n = n.data_ptr()
    a.y = None if y is None else y.data_ptr()
    a.stats = None if stats is None else stats.data_ptr()
    _lib_call("gated_norm_fwd", x.device, C.addressof(a))
    return y, n, stats


class GatedNormFn(torch.autograd.Function):
    """(y, n) of the join, or n alone without a branch."""

    @staticmethod
    def forward(ctx, x, branch, pre_w, post_w, pre_b, post_b, gate, scale, kind, eps, type_):
        _defer.count_uses(*[t for t in (pre_w, post_w, pre_b, post_b, gate) if t is not None])
        a, held, rows = _norm_args(x, branch, pre_w, post_w, pre_b, post_b, gate, scale, kind, eps, type_)
        y, n, stats = _norm_fwd(a, x, branch, rows, True)
        ctx.meta = (scale, kind, eps, type_, rows, x.shape, None if gate is None else gate.shape)
        ctx.gate_kind = a.gate_kind
        ctx.save_for_backward(*held, stats)
        ctx.set_materialize_grads(False)
        return n if branch is None else (y, n)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        xr, br, gr, pre_w, pre_b, post_w, post_b, stats = ctx.saved_tensors
        scale, kind, eps, type_, rows, shape, gshape = ctx.meta
        gk = ctx.gate_kind
        # (saved tensors may come back with other strides: hooks that keep them elsewhere)
        (xr, _, ldx), (br, _, ldb) = _rows(xr), (None, 0, 0) if br is None else _rows(br)
        gr, _, ldg = (gr, 0, 0) if gk != 2 else _rows(gr)
        dy, dn = (None, grads[0]) if br is None else grads
        if dy is None and dn is None:
            return (None,) * 11
        dev, t, width = stats.device, pre_w.dtype, shape[-1]

        def like(p):
            return None if p is None else torch.empty(p.shape, dtype=t, device=dev)

        dy, lddy = (None, 0) if dy is None else _rows(dy)[::2]
        dn, lddn = (None, 0) if dn is None else _rows(dn)[::2]
        dx = torch.empty(shape, dtype=t, device=dev)
        dbr = None if br is None else torch.empty(shape, dtype=t, device=dev)
        dgate = None if gr is None else torch.empty(gshape, dtype=t, device=dev)
        dp = [like(p) for p in (pre_w, pre_b, post_w, post_b)]
        p = [None if s is None else s.data_ptr() for s in (xr, br, gr, pre_w, pre_b, post_w, post_b)]
        a = _NormArgs(type_, kind, gk, width, rows, scale, eps, *p, ldx, ldb, ldg, None, None, stats.data_ptr(),
                      None if dy is None else dy.data_ptr(), None if dn is None else dn.data_ptr(), lddy, lddn,
                      *[None if s is None else s.data_ptr() for s in (dx, dbr, dgate, *dp)])
        ws = _ws(lib.gated_norm_workspace(C.addressof(a)), dev)
        a.workspace = ws.data_ptr()
        _lib_call("gated_norm_bwd", dev, C.addressof(a))
        out = (dx, dbr, dp[0], dp[2], dp[1], dp[3], dgate)
        return tuple(g if n else None for g, n in zip(out, ctx.needs_input_grad)) + (None,) * 4


def _check_norm(x, params, kind, eps):
    if kind not in KINDS:
        raise ValueError("gated_norm: kind is 'rms' or 'layer'")
    if not (eps > 0 and math.isfinite(eps)):
        raise ValueError("gated_norm: eps is a positive number")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= 8192:
        raise ValueError("gated_norm: the last axis has 1 to 8192 channels")
    for name, p in params.items():
        if p is not None and tuple(p.shape) != (x.shape[-1],):
            raise ValueError(f"gated_norm: {name} has {x.shape[-1]} channels as x, not {tuple(p.shape)}")
    if kind == "rms" and (params.get("pre_bias") is not None or params.get("post_bias") is not None):
        raise ValueError("gated_norm: biases belong to kind 'layer'")
    if x.numel() // x.shape[-1] >= 1 << 31:
        raise ValueError("gated_norm: fewer than 2^31 rows")


def gated_norm(x, branch, pre_weight, post_weight, pre_bias=None, post_bias=None, gate=None, residual_scale=1.0,
               kind="rms", eps=1e-5):
    """(y, n) of the join between two blocks (PackedLayers.gated_norm)."""
    type_ = _type_of("gated_norm", x, branch, pre_weight, post_weight, pre_bias, post_bias, gate)
    _check_norm(x, dict(pre_weight=pre_weight, post_weight=post_weight, pre_bias=pre_bias, post_bias=post_bias), kind,
                eps)
    if branch.shape != x.shape:
        raise ValueError(f"gated_norm: branch is {tuple(branch.shape)}, x is {tuple(x.shape)}")
    if gate is not None and gate.shape != x.shape and tuple(gate.shape) != (x.shape[-1],):
        raise ValueError("gated_norm: gate has one value per channel, or x's shape")
    residual_scale = float(residual_scale)
    if not math.isfinite(residual_scale):
        raise ValueError("gated_norm: residual_scale is a finite number")
    args = (x, branch, pre_weight, post_weight, pre_bias, post_bias, gate, residual_scale, KINDS[kind], float(eps),
            type_)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:7]):
        return GatedNormFn.apply(*args)
    a, held, rows = _norm_args(*args)
    return _norm_fwd(a, x, branch, rows, False)[:2]


def pre_norm(x, weight, bias=None, kind="rms", eps=1e-5):
    """The norm alone, before a first block (PackedLayers.pre_norm)."""
    type_ = _type_of("pre_norm", x, weight, bias)
    _check_norm(x, dict(pre_weight=weight, pre_bias=bias), kind, eps)
    args = (x, None, weight, None, bias, None, None, 1.0, KINDS[kind], float(eps), type_)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return GatedNormFn.apply(*args)
    a, held, rows = _norm_args(*args)
    return _norm_fwd(a, x, None, rows, False)[1]


# ---------------------------------------------------------------------------
# activations kept in 8 bits
# ---------------------------------------------------------------------------
class Packed8:
    """A tensor in 8 bits (pack8): `codes` int8 and one power of two for every 32 of them."""
    __slots__ = ("codes", "exponents", "shape", "dtype")

    def __init__(self, codes, exponents, shape, dtype):
        self.codes, self.exponents, self.shape, self.dtype = codes, exponents, shape, dtype


def _codes_for(x):
    n = x.numel()
    return (torch.empty(n, dtype=torch.int8, device=x.device),
            torch.empty((n + 31) // 32, dtype=torch.uint8, device=x.device))


def pack8(x):
    """x in 8 bits: blocks of 32 consecutive values (in memory order of a contiguous x) share a power
    of two (PackedLayers.pack8)."""
    type_ = _type_of("pack8", x)
    x = x.detach().contiguous()
    codes, exps = _codes_for(x)
    _lib_call("pack8", x.device, type_, x.data_ptr(), x.numel(), codes.data_ptr(), exps.data_ptr())
    return Packed8(codes, exps, x.shape, x.dtype)


def unpack8(packed):
    """The values that a Packed8 stands for, in its own shape and type."""
    if not isinstance(packed, Packed8):
        raise TypeError("unpack8: takes what pack8 returns")
    codes, exps, n = packed.codes, packed.exponents, math.prod(packed.shape)
    _lib.require_device(codes, exps)
    if codes.device != exps.device or packed.dtype not in TYPES:
        raise ValueError("unpack8: codes and exponents on one device, of a float32, bfloat16 or float16 tensor")
    if (codes.dtype != torch.int8 or exps.dtype != torch.uint8 or codes.numel() != n or exps.numel() != (n + 31) // 32 or
            not codes.is_contiguous() or not exps.is_contiguous()):
        raise ValueError(f"unpack8: {n} values are {n} int8 codes and {(n + 31) // 32} uint8 exponents, each contiguous")
    return _unpack(packed.codes, packed.exponents, packed.shape, packed.dtype)


def _unpack(codes, exps, shape, dtype):
    out = torch.empty(shape, dtype=dtype, device=codes.device)
    _lib_call("unpack8", codes.device, TYPES[dtype], codes.data_ptr(), exps.data_ptr(), out.numel(), out.data_ptr())
    return out


def _gelu8_fwd(x):
    y = torch.empty_like(x)
    codes, exps = _codes_for(x)
    _lib_call("gelu8_fwd", x.device, TYPES[x.dtype], x.data_ptr(), x.numel(), y.data_ptr(), codes.data_ptr(), exps.data_ptr())
    return y, codes, exps


def _gelu8_bwd(codes, exps, dy, again):
    dx = torch.empty_like(dy)
    y = torch.empty_like(dy) if again else None
    _lib_call("gelu8_bwd", dy.device, TYPES[dy.dtype], codes.data_ptr(), exps.data_ptr(), dy.data_ptr(), dy.numel(), dx.data_ptr(),
                      None if y is None else y.data_ptr())
    return dx, y


class Gelu8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        x = x.contiguous()
        y, codes, exps = _gelu8_fwd(x)
        ctx.save_for_backward(codes, exps)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, exps = ctx.saved_tensors
        return _gelu8_bwd(codes, exps, dy.contiguous(), False)[0]


def gelu8(x):
    """GELU (erf form) that keeps its input in 8 bits for the backward pass (PackedLayers.gelu8)."""
    _type_of("gelu8", x)
    if torch.is_grad_enabled() and x.requires_grad:
        return Gelu8Fn.apply(x)
    return _gelu(x)


def _gelu(x):
    """GELU alone: nothing is kept."""
    x = x.contiguous()
    y = torch.empty_like(x)
    _lib_call("gelu8_fwd", x.device, TYPES[x.dtype], x.data_ptr(), x.numel(), y.data_ptr(), None, None)
    return y


def _own_type():
    """Around the library products of linear8: autocast would give them another type than their tensors'."""
    if torch.is_autocast_enabled("cuda"):
        return torch.autocast("cuda", enabled=False)
    return contextlib.nullcontext()


class Linear8Fn(torch.autograd.Function):
    """act(x) W^T + b that keeps x in 8 bits: the products are the library's, the backward reads the
    kept x once for GELU'(x) and the weight gradient's operand."""

    @staticmethod
    def forward(ctx, x, W, b, act):
        _defer.count_uses(*[t for t in (W, b) if t is not None])
        x = x.contiguous()
        if act:
            y, codes, exps = _gelu8_fwd(x)
        else:
            p = pack8(x)
            y, codes, exps = x, p.codes, p.exponents
        ctx.act, ctx.shape, ctx.has_b = act, x.shape, b is not None
        ctx.save_for_backward(codes, exps, W)
        return torch.nn.functional.linear(y, W, b)

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        with _own_type():
            return Linear8Fn.gradients(ctx, do)

    @staticmethod
    def gradients(ctx, do):
        codes, exps, W = ctx.saved_tensors
        g = do.reshape(math.prod(ctx.shape[:-1]), W.shape[0]).contiguous()
        need = ctx.needs_input_grad
        dx = dW = db = None
        dy = torch.mm(g, W) if (need[0] or ctx.act) else None
        if ctx.act:
            dx, y = _gelu8_bwd(codes, exps, dy, need[1])
        else:
            dx, y = dy, _unpack(codes, exps, (g.shape[0], W.shape[1]), W.dtype) if need[1] else None
        if need[1]:
            dW = torch.mm(g.t(), y)
        if ctx.has_b and need[2]:
            # a product with ones, not torch's sum: that one records memory clears into a captured graph
            db = torch.mv(g.t(), g.new_ones(g.shape[0]))
        return dx.reshape(ctx.shape) if need[0] else None, dW, db, None


def linear8(x, weight, bias=None, act=None):
    """act(x) weight^T + bias, x kept in 8 bits for the backward pass (PackedLayers.linear8)."""
    _type_of("linear8", x, weight, bias)
    if act not in (None, "gelu"):
        raise ValueError("linear8: act is None or 'gelu'")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1] or (bias is not None and tuple(bias.shape) != (weight.shape[0],)):
        raise ValueError("linear8: x [.., in], weight [out, in], bias [out]")
    with _own_type():
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
            return Linear8Fn.apply(x, weight, bias, act == "gelu")
        return torch.nn.functional.linear(_gelu(x) if act else x, weight, bias)
