"""The operators of a bounded cache and of the short convolution (include/sc_ops.h) on the CPU: their structures are the
header's, and every request that they do not take is refused before any HIP call, with its reason."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
FAKE = 1 << 40   # stands for device addresses: every request below is refused before they are used


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


def _same_as_the_header(ops, tmp_path, structs):
    lines = [f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for n, s in structs.items() for f, _ in s._fields_]
    lines += [f'printf("{n} %zu\\n", sizeof({n}));' for n in structs]
    src = tmp_path / "offsets.c"
    src.write_text('#include <stdio.h>\n#include "sc_ops.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-std=c11", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "offsets")], check=True)
    said = dict(x.split() for x in subprocess.run([str(tmp_path / "offsets")], check=True, capture_output=True, text=True).stdout.splitlines())
    for n, s in structs.items():
        assert int(said[n]) == C.sizeof(s), n
        for f, _ in s._fields_:
            assert int(said[f"{n}.{f}"]) == getattr(s, f).offset, (n, f)


def _cache(ops, **kw):
    base = dict(format=0, n_head_kv=2, head_dim=256, page_size=4, n_pages=64, k=FAKE, v=FAKE, table=FAKE, table_ld=64)
    return ops.KvCache(**{**base, **kw})


def _refused(sc, code, why, want=None):
    assert code == (sc.SC_EINVAL if want is None else want), sc.last_error()
    assert why in sc.last_error(), sc.last_error()


# ---- positions of several axes -------------------------------------------------------------------------------------------


def _rope(ops, **kw):
    base = dict(tokens=5, n_seqs=5, cu=None, pos0=FAKE, dtype=1, k=FAKE, v=FAKE, q=FAKE, q_out=FAKE, k_ld=512, v_ld=512,
                q_ld=24 * 256, q_out_ld=24 * 256, n_head=24, pairing=0, rot_dim=64, inv_freq=FAKE)
    return ops.RopeAppendDesc(**{**base, **kw})


def _axes(ops, axis=None, **kw):
    pairs = (C.c_uint8 * 128)(*(axis or [0] * 32))
    a = ops.RopeAxesDesc(**{**dict(n_axes=3, host_axis=C.cast(pairs, C.POINTER(C.c_uint8)), pos=FAKE, pos_ld=5), **kw})
    a.keep = pairs
    return a


def test_axes_structure_matches_the_header(ops, tmp_path):
    _same_as_the_header(ops, tmp_path, {"sc_rope_axes": ops.RopeAxesDesc})


@pytest.mark.parametrize("kw,why", [
    (dict(n_axes=0), "n_axes"), (dict(n_axes=5), "n_axes"), (dict(pos=None), "pos"), (dict(pos=FAKE + 4), "pos"), (dict(pos_ld=4), "pos_ld"),
    (dict(pos_ld=1 << 41), "pos_ld"), (dict(host_axis=None), "host_axis"), (dict(axis=[0] * 31 + [3]), "not below n_axes"),
    (dict(axis=[255] + [0] * 31), "not below n_axes"), (dict(axis=[1] * 32, n_axes=1), "not below n_axes")])
def test_axes_refused(sc, ops, kw, why):
    a = _axes(ops, **kw)
    _refused(sc, sc.lib.sc_rope_axes_append_async(C.byref(_cache(ops)), C.byref(_rope(ops)), C.byref(a), None), why)


@pytest.mark.parametrize("kw,why", [(dict(tokens=6), "one row a sequence"), (dict(pos0=None), "pos0"), (dict(rot_dim=4), "rot_dim"),
                                    (dict(q=None), "n_head"), (dict(k_ld=508), "k_ld")])
def test_appends_with_axes_refused(sc, ops, kw, why):
    _refused(sc, sc.lib.sc_rope_axes_append_async(C.byref(_cache(ops)), C.byref(_rope(ops, **kw)), C.byref(_axes(ops, pos_ld=9)), None), why)


def test_missing_axes_refused(sc, ops):
    c, r, a = _cache(ops), _rope(ops), _axes(ops)
    _refused(sc, sc.lib.sc_rope_axes_append_async(C.byref(c), None, C.byref(a), None), "missing request")
    _refused(sc, sc.lib.sc_rope_axes_append_async(C.byref(c), C.byref(r), None, None), "missing request")
    _refused(sc, sc.lib.sc_rope_axes_append_async(None, C.byref(r), C.byref(a), None), "missing cache")
    _refused(sc, sc.lib.sc_rope_append_async(C.byref(c), C.byref(_rope(ops, rot_dim=4)), None), "rope_append")


def test_nothing_to_turn_needs_no_axes(sc, ops):
    """Without tokens nothing is launched (there is no GPU here), and without rotation no pair has an axis."""
    a = _axes(ops, host_axis=None)
    assert sc.lib.sc_rope_axes_append_async(C.byref(_cache(ops)), C.byref(_rope(ops, tokens=0, cu=FAKE, rot_dim=0)), C.byref(a), None) == sc.SC_OK


def test_axes_of_pairs(ops):
    assert ops.axis_of_pairs((3, 2, 1)) == [0, 0, 0, 1, 1, 2]
    assert ops.axis_of_pairs((3, 2, 1), by_turns=True) == [0, 1, 2, 0, 1, 0]
    kw = dict(n_seqs=1, tokens=1, pos0=FAKE, inv_freq=FAKE, rot_dim=8, pos=FAKE)
    with pytest.raises(ValueError):
        ops.RopeAxesAppend(_cache(ops), FAKE, FAKE, "f32", axis=[0] * 3, n_axes=1, **kw)
    with pytest.raises(ValueError):
        ops.RopeAxesAppend(_cache(ops), FAKE, FAKE, "f32", axis=[0, 0, 0, 300], n_axes=3, **kw)


# ---- the short convolution -----------------------------------------------------------------------------------------------


def _conv(ops, **kw):
    base = dict(channels=8192, taps=4, n_seqs=5, tokens=5, cu=None, dtype=1, x=FAKE, out=2 * FAKE, x_ld=8192, out_ld=8192, weight=FAKE,
                bias=FAKE, activation=1, state=FAKE, state_offset=0, state_layout=0, state_ld=0)
    return ops.ConvDesc(**{**base, **kw})


def test_conv_structure_matches_the_header(ops, tmp_path):
    _same_as_the_header(ops, tmp_path, {"sc_conv": ops.ConvDesc})


@pytest.mark.parametrize("kw,why", [
    (dict(channels=0), "channels"), (dict(channels=12), "channels"), (dict(channels=(1 << 20) + 8), "channels"), (dict(taps=1), "taps"),
    (dict(taps=6), "taps"), (dict(n_seqs=0, tokens=0), "n_seqs"), (dict(n_seqs=4097), "n_seqs"), (dict(tokens=-1, cu=FAKE), "tokens"),
    (dict(tokens=(1 << 23) + 1, cu=FAKE), "tokens"), (dict(tokens=6), "one row a sequence"), (dict(cu=FAKE + 4), "cu"),
    (dict(dtype=2), "dtype"), (dict(x=None), "x and out"), (dict(out=FAKE + 8), "x and out"), (dict(x_ld=8190), "x_ld"),
    (dict(out_ld=8194), "x_ld"), (dict(dtype=0, x_ld=8196), "x_ld"), (dict(x_ld=(1 << 22) + 4), "x_ld"), (dict(weight=None), "weight"),
    (dict(weight=FAKE + 4), "weight"), (dict(bias=FAKE + 8), "bias"), (dict(activation=2), "activation"), (dict(state=None), "state"),
    (dict(state=FAKE + 4), "state"), (dict(state_offset=-4), "state_offset"), (dict(state_offset=6), "state_offset"),
    (dict(state_offset=(1 << 40) + 4), "state_offset"), (dict(state_layout=2), "state_layout"),
    (dict(state_layout=1, state_ld=8188), "state_ld"), (dict(state_layout=1, state_ld=8194), "state_ld"),
    (dict(state_layout=1, state_ld=1 << 41), "state_ld")])
def test_convolutions_refused(sc, ops, kw, why):
    _refused(sc, sc.lib.sc_conv_async(C.byref(_conv(ops, **kw)), None), why)


@pytest.mark.parametrize("kw", [
    dict(cu=FAKE, out=FAKE), dict(cu=FAKE, out=FAKE + 4 * 8192 * 4), dict(out=FAKE, x_ld=8196, out_ld=8192), dict(out=FAKE + 16),
    dict(cu=FAKE, x=FAKE + 8192 * 4 - 16, x_ld=16384, out=FAKE, out_ld=16384)])
def test_outputs_over_inputs_refused(sc, ops, kw):
    _refused(sc, sc.lib.sc_conv_async(C.byref(_conv(ops, **kw)), None), "out must not overlap x")


@pytest.mark.parametrize("kw", [
    dict(out=FAKE), dict(cu=FAKE, out=FAKE + 5 * 8192 * 4), dict(cu=FAKE, out=FAKE + 8192 * 4, x_ld=16384, out_ld=16384),
    dict(bias=None, state_layout=1, state_ld=8192)])
def test_outputs_beside_inputs_taken(sc, ops, kw):
    if sc.device_count() > 0:
        pytest.skip("the addresses are none: only where nothing can be launched")
    assert sc.lib.sc_conv_async(C.byref(_conv(ops, **kw)), None) == sc.SC_EHIP, sc.last_error()


def test_missing_and_empty_convolutions(sc, ops):
    _refused(sc, sc.lib.sc_conv_async(None, None), "missing request")
    assert sc.lib.sc_conv_async(C.byref(_conv(ops, tokens=0, cu=FAKE)), None) == sc.SC_OK


# ---- eviction ------------------------------------------------------------------------------------------------------------


def _evict(ops, **kw):
    base = dict(n_seqs=5, lens=FAKE, max_len=256, keep=100, sinks=4, recent=16, mass=FAKE, mass_out=FAKE, born=FAKE, born_out=FAKE, ld=256,
                known=FAKE, total=FAKE, lens_out=FAKE)
    return ops.KvEvictDesc(**{**base, **kw})


def test_evict_structure_matches_the_header(ops, tmp_path):
    _same_as_the_header(ops, tmp_path, {"sc_kv_evict": ops.KvEvictDesc})


BYTES = 5 * 2 * 256 * 4


@pytest.mark.parametrize("kw,why", [
    (dict(n_seqs=0), "n_seqs"), (dict(n_seqs=1025), "n_seqs"), (dict(max_len=-1), "max_len"), (dict(max_len=257, ld=300), "max_len"),
    (dict(keep=0), "keep"), (dict(keep=1 << 31), "keep"), (dict(sinks=-1), "sinks"), (dict(recent=-1), "recent"), (dict(recent=97), "recent"),
    (dict(sinks=1 << 62, recent=1 << 62), "sinks"), (dict(lens=None), "lens"), (dict(lens_out=None), "lens"), (dict(lens_out=FAKE + 4), "lens"),
    (dict(known=FAKE + 4), "known"), (dict(total=FAKE + 2), "total"), (dict(mass=None), "mass"), (dict(mass_out=None), "mass"),
    (dict(mass_out=FAKE + 2), "mass"), (dict(born=FAKE + 2), "born"), (dict(born=None), "together"), (dict(known=None), "together"),
    (dict(ld=255), "ld"), (dict(ld=1 << 31), "ld"), (dict(max_len=0, ld=0), "ld"), (dict(mass_out=FAKE + BYTES - 4), "share no byte"),
    (dict(mass_out=FAKE - BYTES + 4), "share no byte"), (dict(born_out=FAKE + 4), "share no byte")])
def test_evictions_refused(sc, ops, kw, why):
    c, e = _cache(ops), _evict(ops, **kw)
    _refused(sc, sc.lib.sc_kv_evict_async(C.byref(c), C.byref(e), FAKE, 1 << 50, None), why)
    assert sc.lib.sc_kv_evict_workspace_bytes(C.byref(c), C.byref(e)) == 0


def test_evictions_without_what_they_need(sc, ops):
    c, e = _cache(ops), _evict(ops)
    _refused(sc, sc.lib.sc_kv_evict_async(C.byref(c), None, FAKE, 1 << 40, None), "missing request")
    _refused(sc, sc.lib.sc_kv_evict_async(None, C.byref(e), FAKE, 1 << 40, None), "missing cache")
    _refused(sc, sc.lib.sc_kv_evict_async(C.byref(_cache(ops, format=2)), C.byref(e), FAKE, 1 << 40, None), "format")
    need = sc.lib.sc_kv_evict_workspace_bytes(C.byref(c), C.byref(e))
    assert need > 0
    for ws, n in ((None, need), (FAKE + 8, need), (FAKE, need - 1)):
        _refused(sc, sc.lib.sc_kv_evict_async(C.byref(c), C.byref(e), ws, n, None), "workspace")
    assert sc.lib.sc_kv_evict_workspace_bytes(C.byref(c), C.byref(_evict(ops, keep=256))) > 0   # nothing can be evicted
    assert sc.lib.sc_kv_evict_workspace_bytes(C.byref(c), C.byref(_evict(ops, mass_out=FAKE + BYTES, born_out=FAKE - BYTES))) == need


# ---- mass ----------------------------------------------------------------------------------------------------------------


def _mass(ops, **kw):
    base = dict(n_seqs=5, lens=FAKE, max_len=256, window=0, rows=1, dtype=0, n_head=24, q=FAKE, q_ld=24 * 256, lse=FAKE, scale=0.0625,
                decay=1.0, mass=FAKE, mass_ld=256)
    return ops.AttnMassDesc(**{**base, **kw})


def test_mass_structure_matches_the_header(ops, tmp_path):
    _same_as_the_header(ops, tmp_path, {"sc_attn_mass": ops.AttnMassDesc})


@pytest.mark.parametrize("kw,why", [
    (dict(n_seqs=0), "n_seqs"), (dict(n_seqs=1025), "n_seqs"), (dict(max_len=-1), "max_len"), (dict(max_len=257, mass_ld=300), "max_len"),
    (dict(window=-1), "window"), (dict(dtype=3), "dtype"), (dict(n_head=25), "n_head"), (dict(n_head=0), "n_head"), (dict(rows=0), "rows"),
    (dict(rows=86), "rows"), (dict(rows=1 << 60), "rows"), (dict(n_head=4096, q_ld=4096 * 256), "rows"), (dict(lens=None), "lens"),
    (dict(lens=FAKE + 4), "lens"), (dict(q=None), "q must"), (dict(q=FAKE + 8), "q must"), (dict(q_ld=24 * 256 - 8), "q_ld"),
    (dict(q_ld=24 * 256 + 4), "q_ld"), (dict(lse=FAKE + 2), "lse"), (dict(decay=float("nan")), "decay"), (dict(decay=float("inf")), "decay"),
    (dict(mass=None), "mass"), (dict(mass=FAKE + 2), "mass"), (dict(mass_ld=255), "mass_ld"), (dict(mass_ld=1 << 31), "mass_ld")])
def test_masses_refused(sc, ops, kw, why):
    c, m = _cache(ops), _mass(ops, **kw)
    _refused(sc, sc.lib.sc_attn_mass_async(C.byref(c), C.byref(m), FAKE, 1 << 50, None), why)
    assert sc.lib.sc_attn_mass_workspace_bytes(C.byref(c), C.byref(m)) == 0


def test_masses_without_what_they_need(sc, ops):
    c = _cache(ops)
    _refused(sc, sc.lib.sc_attn_mass_async(C.byref(c), None, FAKE, 1 << 40, None), "missing request")
    _refused(sc, sc.lib.sc_attn_mass_async(None, C.byref(_mass(ops)), FAKE, 1 << 40, None), "missing cache")
    for lse in (FAKE, None):
        m = _mass(ops, lse=lse, rows=85)
        need = sc.lib.sc_attn_mass_workspace_bytes(C.byref(c), C.byref(m))
        assert need > 0
        for ws, n in ((None, need), (FAKE + 8, need), (FAKE, need - 1)):
            _refused(sc, sc.lib.sc_attn_mass_async(C.byref(c), C.byref(m), ws, n, None), "workspace")
    assert sc.lib.sc_attn_mass_async(C.byref(c), C.byref(_mass(ops, max_len=0)), FAKE, 16, None) == sc.SC_OK
