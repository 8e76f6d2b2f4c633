"""The slot that a conversation with a bounded cache is resumed into (examples/bounded_conversation.py): it has room for the cells
that may be kept and the tokens up to the next eviction, whatever the prompt's length was, and the calls made over it say so."""
import sys
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

GEO = dict(n_layers=4, qsa_interval=4, n_head_kv=2, head_dim=128, page_size=4, ssm_state_size=64, ssm_k_heads=2, ssm_v_heads=4,
           ssm_conv_channels=512)
HEADS, EVERY, NEW = 4, 3, 7


@pytest.fixture(scope="module")
def example():
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "strata-concurrent_amd" / "examples"))
    import bounded_conversation
    return bounded_conversation


# prompts longer than what is kept, shorter, and one that no eviction has cut before its hand-off
@pytest.mark.parametrize("prompt,keep,cut,cells", [(150, 40, True, 44), (30, 41, True, 44), (90, 40, False, 96)])
def test_the_resumed_slot(sc, example, cuda, prompt, keep, cut, cells):
    geo = sc.geometry(**GEO)
    b = example.Bounded(geo, HEADS, keep, prompt, EVERY)
    b.prompt(example.Inputs(geo, prompt, HEADS, 1), example.positions(0, prompt - 12, (3, 4), 0), 5)
    width = b.max_cells
    assert width == geo.cells(max(prompt, keep) + EVERY) == b.mass[0].shape[2]   # tokens come before an eviction here too
    if cut:
        b.evict(b.evictions())
    b.hand_off()
    assert b.max_cells == cells == b.slot.max_cells
    assert b.slot.k_pool[0].nbytes == cells * geo.n_head_kv * geo.head_dim * 2
    dec, evictions = example.Decoder(b, example.Inputs(geo, NEW, HEADS, 2)), b.evictions()
    assert {c.desc.max_len for c in [*evictions, *(c for c in dec.calls if hasattr(c.desc, "max_len"))]} == {cells}
    assert {c.desc.ld for c in evictions} == {width} == {c.desc.mass_ld for c in dec.calls if hasattr(c.desc, "mass_ld")}
    for t in range(NEW):
        dec.token(t, prompt + t)
        if (t + 1) % EVERY == 0:
            b.evict(evictions)
        sc.device_sync()
        assert b.cells <= cells
        # nothing is left behind the cells that there are
        mass = b.mass[0].numpy().reshape(geo.n_head_kv, width)
        assert np.isfinite(mass).all() and not mass[:, b.cells:].any()
        assert all(np.isfinite(o.numpy()).all() for o in dec.attn_out)
