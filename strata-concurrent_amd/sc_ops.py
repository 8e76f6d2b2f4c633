"""Python binding of include/sc_ops.h (libsc_handoff.so): the operators that run on a decode slot between two hand-offs.

Each class is one layer's call with its device buffers (anything with `data_ptr()`, or raw pointers) and its workspace;
`launch()` enqueues it and nothing else.  Lengths, positions, page tables and states are read when the kernels run, so one
object serves every step of a batch."""
from __future__ import annotations

import ctypes as C

import sc_handoff as sc
from sc_handoff import lib

SC_ROPE_HALVES, SC_ROPE_NEIGHBOURS = 0, 1
ATTN_MAX_SEQS = 1024

_P, _I64, _U64, _I32 = C.c_void_p, C.c_int64, C.c_uint64, C.c_int32


class KvCache(C.Structure):
    """sc_kv_cache: one layer's paged K and V of many sequences."""
    _fields_ = [("format", _I32), ("n_head_kv", _I64), ("head_dim", _I64), ("page_size", _I64), ("n_pages", _I64),
                ("k", _P), ("v", _P), ("k_scale", _P), ("v_scale", _P), ("table", _P), ("table_ld", _I64)]


class RopeAppendDesc(C.Structure):
    _fields_ = [("tokens", _I64), ("n_seqs", _I32), ("cu", _P), ("pos0", _P), ("dtype", _I32), ("k", _P), ("v", _P),
                ("q", _P), ("q_out", _P), ("k_ld", _I64), ("v_ld", _I64), ("q_ld", _I64), ("q_out_ld", _I64),
                ("n_head", _I64), ("pairing", _I32), ("rot_dim", _I64), ("inv_freq", _P)]


class AttnDecodeDesc(C.Structure):
    _fields_ = [("n_seqs", _I32), ("lens", _P), ("max_len", _I64), ("window", _I64), ("dtype", _I32), ("n_head", _I64),
                ("q", _P), ("out", _P), ("q_ld", _I64), ("out_ld", _I64), ("lse", _P), ("scale", C.c_float)]


class GdnDesc(C.Structure):
    _fields_ = [("k_heads", _I64), ("v_heads", _I64), ("state_size", _I64), ("n_seqs", _I32), ("tokens", _I64), ("cu", _P),
                ("dtype", _I32), ("q", _P), ("k", _P), ("v", _P), ("out", _P), ("q_ld", _I64), ("k_ld", _I64),
                ("v_ld", _I64), ("out_ld", _I64), ("g", _P), ("beta", _P), ("gate_ld", _I64), ("scale", C.c_float),
                ("l2norm", _I32), ("eps", C.c_float), ("state", _P), ("state_offset", _I64), ("state_head_ld", _I64),
                ("state_key_ld", _I64)]


_SIGS = {
    "sc_rope_append_async": (C.c_int, [C.POINTER(KvCache), C.POINTER(RopeAppendDesc), _P]),
    "sc_attn_decode_workspace_bytes": (_U64, [C.POINTER(KvCache), C.POINTER(AttnDecodeDesc)]),
    "sc_attn_decode_async": (C.c_int, [C.POINTER(KvCache), C.POINTER(AttnDecodeDesc), _P, _U64, _P]),
    "sc_gdn_step_async": (C.c_int, [C.POINTER(GdnDesc), _P]),
    "sc_gdn_chunk_workspace_bytes": (_U64, [C.POINTER(GdnDesc)]),
    "sc_gdn_chunk_async": (C.c_int, [C.POINTER(GdnDesc), _P, _U64, _P]),
}
for _name, (_res, _args) in _SIGS.items():
    _fn = getattr(lib, _name)
    _fn.restype = _res
    _fn.argtypes = _args

EXPORTS = tuple(_SIGS)

_DTYPES = {"f16": sc.SC_DTYPE_F16, "f32": sc.SC_DTYPE_F32, sc.SC_DTYPE_F16: sc.SC_DTYPE_F16, sc.SC_DTYPE_F32: sc.SC_DTYPE_F32}
_PAIRS = {"halves": SC_ROPE_HALVES, "neighbours": SC_ROPE_NEIGHBOURS}


def _ptr(x) -> int | None:
    return x if x is None or isinstance(x, int) else x.data_ptr()


def _dtype(x) -> int:
    if x not in _DTYPES:
        raise ValueError(f"activations are 'f16' or 'f32', not {x!r}")
    return _DTYPES[x]


def kv_cache(k, v, k_scale=None, v_scale=None, *, n_pages: int, n_head_kv: int, head_dim: int, page_size: int, table=None,
             table_ld: int) -> KvCache:
    """One layer's paged cache: f16 pools, or int8 codes when the scale pools are given.  The buffers stay the caller's
    and must outlive the operators made with it."""
    c = KvCache(format=sc.SC_KV_INT8 if k_scale is not None else sc.SC_KV_F16, n_head_kv=n_head_kv, head_dim=head_dim,
                page_size=page_size, n_pages=n_pages, k=_ptr(k), v=_ptr(v), k_scale=_ptr(k_scale), v_scale=_ptr(v_scale),
                table=_ptr(table), table_ld=table_ld)
    c.keep = (k, v, k_scale, v_scale, table)
    return c


def slot_cache(geo: sc.Geometry, slot: sc.Slot, layer: int) -> KvCache:
    """QSA layer `layer` of an f16 decode slot (sc_handoff.Slot): what a carve or a resume has filled."""
    table = slot.tables[layer] if slot.tables else None
    return kv_cache(slot.k_pool[layer], slot.v_pool[layer], n_pages=slot.n_pages, n_head_kv=geo.n_head_kv,
                    head_dim=geo.head_dim, page_size=geo.page_size, table=table, table_ld=slot.max_cells // geo.page_size)


class _Op:
    """A call with everything it was made from; the C structures are built once."""

    def _keep(self, *things) -> None:
        self._things = things

    def launch(self, stream=None) -> None:
        code = self._call(*self._args, stream if stream is None or isinstance(stream, int) else stream.handle)
        if code:
            raise sc.ScError(code, self._name)


class RopeAppend(_Op):
    """Rows of new tokens into a paged cache, keys and queries rotated (sc_rope_append_async)."""
    _name, _call = "sc_rope_append_async", staticmethod(lib.sc_rope_append_async)

    def __init__(self, cache: KvCache, k, v, act, *, n_seqs: int, tokens: int, pos0, inv_freq=None, rot_dim: int = 0,
                 pairs="halves", cu=None, q=None, q_out=None, n_head: int = 0, k_ld: int | None = None,
                 v_ld: int | None = None, q_ld: int | None = None, q_out_ld: int | None = None):
        row, q_row = cache.n_head_kv * cache.head_dim, n_head * cache.head_dim
        self.desc = RopeAppendDesc(
            tokens=tokens, n_seqs=n_seqs, cu=_ptr(cu), pos0=_ptr(pos0), dtype=_dtype(act), k=_ptr(k), v=_ptr(v), q=_ptr(q),
            q_out=_ptr(q_out), k_ld=row if k_ld is None else k_ld, v_ld=row if v_ld is None else v_ld,
            q_ld=q_row if q_ld is None else q_ld, q_out_ld=q_row if q_out_ld is None else q_out_ld, n_head=n_head,
            pairing=_PAIRS.get(pairs, pairs), rot_dim=rot_dim, inv_freq=_ptr(inv_freq))
        self._keep(cache, k, v, q, q_out, cu, pos0, inv_freq)
        self._args = (C.byref(cache), C.byref(self.desc))


class AttnDecode(_Op):
    """One new token a sequence over its paged cache (sc_attn_decode_async).  `max_len` bounds every length; a workspace
    is allocated here unless one is given (`workspace`, `workspace_bytes`)."""
    _name, _call = "sc_attn_decode_async", staticmethod(lib.sc_attn_decode_async)

    def __init__(self, cache: KvCache, q, out, act, *, n_seqs: int, n_head: int, lens, max_len: int, scale: float,
                 window: int = 0, lse=None, q_ld: int | None = None, out_ld: int | None = None, workspace=None,
                 workspace_bytes: int = 0):
        row = n_head * cache.head_dim
        self.desc = AttnDecodeDesc(n_seqs=n_seqs, lens=_ptr(lens), max_len=max_len, window=window, dtype=_dtype(act),
                                   n_head=n_head, q=_ptr(q), out=_ptr(out), q_ld=row if q_ld is None else q_ld,
                                   out_ld=row if out_ld is None else out_ld, lse=_ptr(lse), scale=scale)
        if workspace is None:
            workspace_bytes = int(lib.sc_attn_decode_workspace_bytes(C.byref(cache), C.byref(self.desc)))
            if not workspace_bytes:
                raise sc.ScError(sc.SC_EINVAL, "sc_attn_decode_workspace_bytes")
            workspace = sc.DeviceBuffer(workspace_bytes, "uint8")
        self._keep(cache, q, out, lens, lse, workspace)
        self._args = (C.byref(cache), C.byref(self.desc), _ptr(workspace), workspace_bytes)


class GdnStates:
    """Where the recurrent states of a batch lie: the bases, device array of one pointer a sequence, and the strides."""

    def __init__(self, bases, v_heads: int, state_size: int, offset: int, head_ld: int, key_ld: int, keep=()):
        self.bases = sc.DeviceBuffer(max(len(bases), 1), "uint64")
        self.bases.upload([b or 0 for b in bases])
        self.n_seqs, self.v_heads, self.state_size = len(bases), v_heads, state_size
        self.offset, self.head_ld, self.key_ld, self.keep = offset, head_ld, key_ld, keep


def _strides(layout: str, v_heads: int, state_size: int) -> tuple[int, int]:
    """(floats between heads, floats between keys): a slot's row (S, HV, S), or the prefill layout [HV][S][S]."""
    try:
        return {"slot": (state_size, v_heads * state_size), "prefill": (state_size * state_size, state_size)}[layout]
    except KeyError:
        raise ValueError(f"a state's layout is 'slot' or 'prefill', not {layout!r}") from None


def gdn_states(state, *, n_seqs: int, v_heads: int, state_size: int, layout: str = "slot") -> GdnStates:
    """States of one layer, one after the other in one f32 buffer."""
    base, each = _ptr(state), 4 * v_heads * state_size * state_size
    return GdnStates([base + i * each for i in range(n_seqs)], v_heads, state_size, 0, *_strides(layout, v_heads, state_size),
                     keep=state)


def slot_states(geo: sc.Geometry, slots, layer: int) -> GdnStates:
    """GDN layer `layer` of decode slots (sc_handoff.Slot, or None for a sequence without one)."""
    bases = [None if s is None else s.gdn.data_ptr() for s in slots]
    return GdnStates(bases, geo.ssm_v_heads, geo.ssm_state_size, layer * geo.gdn_row_floats,
                     *_strides("slot", geo.ssm_v_heads, geo.ssm_state_size), keep=slots)


class _Gdn(_Op):
    def __init__(self, states: GdnStates, q, k, v, g, beta, out, act, *, k_heads: int, n_seqs: int, tokens: int, cu=None,
                 scale: float, l2norm: bool = False, eps: float = 1e-6, q_ld: int | None = None, k_ld: int | None = None,
                 v_ld: int | None = None, out_ld: int | None = None, gate_ld: int | None = None):
        row, v_row = k_heads * states.state_size, states.v_heads * states.state_size
        if n_seqs != states.n_seqs:
            raise ValueError(f"{n_seqs} sequences with the states of {states.n_seqs}")
        self.desc = GdnDesc(
            k_heads=k_heads, v_heads=states.v_heads, state_size=states.state_size, n_seqs=n_seqs, tokens=tokens,
            cu=_ptr(cu), dtype=_dtype(act), q=_ptr(q), k=_ptr(k), v=_ptr(v), out=_ptr(out),
            q_ld=row if q_ld is None else q_ld, k_ld=row if k_ld is None else k_ld, v_ld=v_row if v_ld is None else v_ld,
            out_ld=v_row if out_ld is None else out_ld, g=_ptr(g), beta=_ptr(beta),
            gate_ld=states.v_heads if gate_ld is None else gate_ld, scale=scale, l2norm=int(l2norm), eps=eps,
            state=_ptr(states.bases), state_offset=states.offset, state_head_ld=states.head_ld,
            state_key_ld=states.key_ld)
        self._keep(states, q, k, v, g, beta, out, cu)


class GdnStep(_Gdn):
    """The gated delta rule for one token of every sequence (sc_gdn_step_async)."""
    _name, _call = "sc_gdn_step_async", staticmethod(lib.sc_gdn_step_async)

    def __init__(self, states, q, k, v, g, beta, out, act, **kw):
        super().__init__(states, q, k, v, g, beta, out, act, **{**kw, "cu": None})
        self._args = (C.byref(self.desc),)


class GdnChunk(_Gdn):
    """The gated delta rule over every sequence's tokens (sc_gdn_chunk_async); a workspace is allocated here unless one is
    given."""
    _name, _call = "sc_gdn_chunk_async", staticmethod(lib.sc_gdn_chunk_async)

    def __init__(self, states, q, k, v, g, beta, out, act, *, workspace=None, workspace_bytes: int = 0, **kw):
        super().__init__(states, q, k, v, g, beta, out, act, **kw)
        if workspace is None:
            workspace_bytes = int(lib.sc_gdn_chunk_workspace_bytes(C.byref(self.desc)))
            if not workspace_bytes:
                raise sc.ScError(sc.SC_EINVAL, "sc_gdn_chunk_workspace_bytes")
            workspace = sc.DeviceBuffer(workspace_bytes, "uint8")
        self._workspace = workspace
        self._args = (C.byref(self.desc), _ptr(workspace), workspace_bytes)
