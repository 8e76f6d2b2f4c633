"""include/sc_ops.h on the CPU: the library exports what the header declares, and every request that an operator does not
take is refused before any HIP call, with its reason."""
import ctypes as C
import re
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
FAKE = 1 << 40   # stands for device addresses: every request below is refused before they are used


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


def test_library_exports_every_declared_symbol(sc, ops):
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "sc_ops.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b(sc_[a-z0-9_]+)\s*\(", text))
    assert names == set(ops.EXPORTS)
    for name in names:
        assert hasattr(sc.lib, name), name


def test_structures_match_the_header(ops, tmp_path):
    """The binding's structures have the header's sizes and offsets, as a C compiler lays them out."""
    import subprocess
    structs = {"sc_kv_cache": ops.KvCache, "sc_rope_append": ops.RopeAppendDesc, "sc_attn_decode": ops.AttnDecodeDesc,
               "sc_gdn": ops.GdnDesc}
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


INT8 = dict(format=1, k_scale=FAKE, v_scale=FAKE)
CACHE_REFUSALS = [(dict(format=2), "format"), (dict(format=3), "format"), (dict(head_dim=96), "head_dim"),
                  (dict(n_head_kv=0), "n_head_kv"), (dict(n_head_kv=257), "n_head_kv"), (dict(page_size=0), "page_size"),
                  (dict(page_size=65537), "page_size"), (dict(n_pages=0), "n_pages"), (dict(n_pages=1 << 31), "n_pages"),
                  (dict(table_ld=0), "table_ld"), (dict(table_ld=1 << 30), "table_ld"), (dict(k=None), "pools"),
                  (dict(v=FAKE + 8), "pools"), (dict(INT8, k_scale=None), "scale"), (dict(INT8, v_scale=FAKE + 4), "scale"),
                  (dict(table=FAKE + 2), "table"), (dict(table=None, table_ld=(1 << 29) - 1, n_pages=1), "identity")]


def _refused(sc, code, why, want=None):
    assert code == (sc.SC_EINVAL if want is None else want), sc.last_error()
    assert why in sc.last_error(), sc.last_error()


def _rope(ops, **kw):
    base = dict(tokens=5, n_seqs=5, cu=None, pos0=FAKE, dtype=1, k=FAKE, v=FAKE, q=FAKE, q_out=FAKE, k_ld=512, v_ld=512,
                q_ld=24 * 256, q_out_ld=24 * 256, n_head=24, pairing=0, rot_dim=64, inv_freq=FAKE)
    return ops.RopeAppendDesc(**{**base, **kw})


def _attn(ops, **kw):
    base = dict(n_seqs=5, lens=FAKE, max_len=256, window=0, dtype=0, n_head=24, q=FAKE, out=FAKE, q_ld=24 * 256,
                out_ld=24 * 256, lse=FAKE, scale=0.0625)
    return ops.AttnDecodeDesc(**{**base, **kw})


def _gdn(ops, **kw):
    base = dict(k_heads=16, v_heads=32, state_size=128, n_seqs=5, tokens=5, cu=None, dtype=1, q=FAKE, k=FAKE, v=FAKE,
                out=FAKE, q_ld=2048, k_ld=2048, v_ld=4096, out_ld=4096, g=FAKE, beta=FAKE, gate_ld=32, scale=0.1, l2norm=1,
                eps=1e-6, state=FAKE, state_offset=0, state_head_ld=128, state_key_ld=4096)
    return ops.GdnDesc(**{**base, **kw})


@pytest.mark.parametrize("kw,why", CACHE_REFUSALS)
def test_caches_refused(sc, ops, kw, why):
    c, n = _cache(ops, **kw), 5
    want = sc.SC_ERANGE if why == "identity" else sc.SC_EINVAL
    _refused(sc, sc.lib.sc_rope_append_async(C.byref(c), C.byref(_rope(ops, n_seqs=n)), None), why, want)
    _refused(sc, sc.lib.sc_attn_decode_async(C.byref(c), C.byref(_attn(ops, n_seqs=n)), FAKE, 1 << 40, None), why, want)
    assert sc.lib.sc_attn_decode_workspace_bytes(C.byref(c), C.byref(_attn(ops))) == 0


@pytest.mark.parametrize("kw,why", [
    (dict(n_seqs=0, tokens=0), "n_seqs"), (dict(n_seqs=4097), "n_seqs"), (dict(tokens=-1, cu=FAKE), "tokens"),
    (dict(tokens=(1 << 23) + 1, cu=FAKE), "tokens"), (dict(tokens=6), "one row a sequence"), (dict(pos0=None), "pos0"),
    (dict(cu=FAKE + 4), "cu"), (dict(dtype=2), "dtype"), (dict(k=None), "k and v"), (dict(v=FAKE + 8), "k and v"),
    (dict(k_ld=508), "k_ld"), (dict(v_ld=514), "k_ld"), (dict(dtype=0, k_ld=516), "k_ld"), (dict(q=None), "n_head"),
    (dict(n_head=0), "n_head"), (dict(q_out=None), "q_out"), (dict(q_ld=100), "q_ld"), (dict(q_out_ld=24 * 256 + 4), "one stride"),
    (dict(pairing=2), "pairing"), (dict(rot_dim=4), "rot_dim"), (dict(rot_dim=264), "rot_dim"), (dict(inv_freq=None), "inv_freq")])
def test_appends_refused(sc, ops, kw, why):
    _refused(sc, sc.lib.sc_rope_append_async(C.byref(_cache(ops)), C.byref(_rope(ops, **kw)), None), why)


@pytest.mark.parametrize("kw,why", [
    (dict(n_seqs=0), "n_seqs"), (dict(n_seqs=1025), "n_seqs"), (dict(max_len=-1), "max_len"), (dict(max_len=257), "max_len"),
    (dict(window=-1), "window"), (dict(dtype=3), "dtype"), (dict(n_head=25), "n_head"), (dict(n_head=0), "n_head"),
    (dict(lens=None), "lens"), (dict(q=None), "q and out"), (dict(out=FAKE + 8), "q and out"), (dict(q_ld=24 * 256 - 8), "q_ld"),
    (dict(out_ld=24 * 256 + 4), "q_ld"), (dict(lse=FAKE + 2), "lse")])
def test_attention_refused(sc, ops, kw, why):
    c, a = _cache(ops), _attn(ops, **kw)
    _refused(sc, sc.lib.sc_attn_decode_async(C.byref(c), C.byref(a), FAKE, 1 << 40, None), why)
    assert sc.lib.sc_attn_decode_workspace_bytes(C.byref(c), C.byref(a)) == 0


@pytest.mark.parametrize("kw,why", [
    (dict(state_size=96), "state_size"), (dict(v_heads=33), "v_heads"), (dict(k_heads=0), "v_heads"), (dict(v_heads=1040), "v_heads"),
    (dict(n_seqs=0, tokens=0), "n_seqs"), (dict(tokens=-1), "tokens"), (dict(tokens=4), "one row a sequence"),
    (dict(cu=FAKE), "no cu"), (dict(dtype=2), "dtype"), (dict(q=None), "q, k, v"), (dict(v=FAKE + 4), "q, k, v"),
    (dict(q_ld=2046), "row strides"), (dict(out_ld=4000), "row strides"), (dict(g=None), "g and beta"),
    (dict(gate_ld=31), "g and beta"), (dict(state=None), "state"), (dict(state=FAKE + 4), "state"),
    (dict(state_offset=2), "strides"), (dict(state_head_ld=64), "strides"), (dict(state_key_ld=4090), "strides"),
    (dict(state_head_ld=132), "overlap"), (dict(state_key_ld=2048), "overlap"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps")])
def test_steps_refused(sc, ops, kw, why):
    _refused(sc, sc.lib.sc_gdn_step_async(C.byref(_gdn(ops, **kw)), None), why)
    if why not in ("no cu", "one row a sequence"):
        a = _gdn(ops, **{**kw, "cu": FAKE})
        _refused(sc, sc.lib.sc_gdn_chunk_async(C.byref(a), FAKE, 1 << 40, None), why)
        assert sc.lib.sc_gdn_chunk_workspace_bytes(C.byref(a)) == 0


def test_missing_requests_and_workspaces_refused(sc, ops):
    c, a, g = _cache(ops), _attn(ops), _gdn(ops, cu=FAKE)
    _refused(sc, sc.lib.sc_rope_append_async(C.byref(c), None, None), "missing request")
    _refused(sc, sc.lib.sc_rope_append_async(None, C.byref(_rope(ops)), None), "missing cache")
    _refused(sc, sc.lib.sc_attn_decode_async(C.byref(c), None, FAKE, 1 << 40, None), "missing request")
    _refused(sc, sc.lib.sc_gdn_step_async(None, None), "missing request")
    _refused(sc, sc.lib.sc_gdn_chunk_async(C.byref(_gdn(ops)), FAKE, 1 << 40, None), "cu")
    need = sc.lib.sc_attn_decode_workspace_bytes(C.byref(c), C.byref(a))
    assert need > 0
    for ws, n in ((None, need), (FAKE + 8, need), (FAKE, need - 1)):
        _refused(sc, sc.lib.sc_attn_decode_async(C.byref(c), C.byref(a), ws, n, None), "workspace")
    need = sc.lib.sc_gdn_chunk_workspace_bytes(C.byref(g))
    assert need > 0
    for ws, n in ((None, need), (FAKE + 16, need), (FAKE, need - 1)):
        _refused(sc, sc.lib.sc_gdn_chunk_async(C.byref(g), ws, n, None), "workspace")


def test_nothing_to_do_launches_nothing(sc, ops):
    """A batch without tokens is no error and no launch (there is no GPU here)."""
    assert sc.lib.sc_rope_append_async(C.byref(_cache(ops)), C.byref(_rope(ops, tokens=0, cu=FAKE)), None) == sc.SC_OK
    a = _gdn(ops, tokens=0, cu=FAKE)
    assert sc.lib.sc_gdn_chunk_async(C.byref(a), FAKE, 1 << 40, None) == sc.SC_OK


def test_binding_refuses_unknown_words(ops):
    with pytest.raises(ValueError):
        ops.gdn_states(FAKE, n_seqs=1, v_heads=1, state_size=64, layout="rows")
    with pytest.raises(ValueError):
        ops.AttnDecode(_cache(ops), FAKE, FAKE, "bf16", n_seqs=1, n_head=2, lens=FAKE, max_len=1, scale=1.0)
