"""sc_attn_mass_async over a sequence of more than 2^30 cells, whose pages are one physical page but for the last two: more cells
than one launch has threads for.  The window is short, so that only the last cells have a weight; the others keep their mass, or
half of it.  Tolerances as in test_gpu_mass.py."""
import numpy as np
import pytest

from ops_cases import act, upload

pytestmark = pytest.mark.gpu

PS, D, HEADS, ROWS, WINDOW = 65536, 256, 17, 2, 300
CELLS = (1 << 30) + PS + 70


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


@pytest.mark.parametrize("given", [True, False], ids=["given", "formed"])
def test_more_cells_than_a_launch_has_threads(sc, ops, cuda, given):
    from oracle import sc_ops as plain
    rng, ld = np.random.default_rng(2), -(-CELLS // PS)
    k = rng.standard_normal((3 * PS, D)).astype(np.float16)
    table = np.zeros((1, ld), np.int32)
    table[0, -2:] = 1, 2
    dk = upload(sc, k)
    cache = ops.kv_cache(dk, dk, n_pages=3, n_head_kv=1, head_dim=D, page_size=PS, table=upload(sc, table), table_ld=ld)
    q, q64 = act(rng.standard_normal((ROWS, HEADS, D)), "f16")
    scale = float(np.float32(D ** -0.5))
    span = WINDOW + ROWS   # the last cells
    cells = np.arange(CELLS - span, CELLS)
    K = k[table[0, cells // PS] * PS + cells % PS].astype(np.float64)
    lse, seen = np.zeros((ROWS, HEADS), np.float32), []
    for r in range(ROWS):
        ends = span - ROWS + 1 + r
        seen.append(slice(ends - WINDOW, ends))
        for i in range(HEADS):
            s = scale * K[seen[r]] @ q64[r, i]
            lse[r, i] = np.log(np.exp(s - s.max()).sum()) + s.max()
    want, near = np.zeros(span), np.zeros(span)
    for r in range(ROWS):
        for i in range(HEADS):
            p = plain.attention_mass(q64[r, i], K[seen[r]], scale, float(lse[r, i]) if given else None)
            e = 2.0 ** -19 * scale * np.abs(K[seen[r]] * q64[r, i]).sum(-1).max()
            want[seen[r]] += p
            near[seen[r]] += p * (2 * e + 2.0 ** -20 + ROWS * HEADS * 2.0 ** -24) + 2.0 ** -120
    mass = sc.DeviceBuffer((1, 1, CELLS + 2), "float32")
    places = [0, 128, (1 << 29) - 64, (1 << 29) + 64, (1 << 30) - 64, (1 << 30), (1 << 30) + 1024, CELLS - span]
    old = rng.random((len(places), span)).astype(np.float32)
    mass.fill(0)
    sc.device_sync()
    for at, values in zip(places, old):
        mass.upload(values, at)
    mass.upload(np.full(2, 7.0, np.float32), CELLS)
    print("launching", flush=True)
    ops.AttnMass(cache, upload(sc, q), mass, "f16", n_seqs=1, n_head=HEADS, rows=ROWS, lens=upload(sc, np.array([CELLS])), max_len=CELLS, scale=scale,
                 window=WINDOW, lse=upload(sc, lse) if given else None, decay=0.5, mass_ld=CELLS + 2).launch()
    sc.device_sync()
    for at, values in zip(places[:-1], old):
        upto = min([p for p in places if p > at] + [at + span]) - at   # what the next place's values have not taken
        got = mass.numpy(min(span, upto), at)
        assert np.array_equal(got, 0.5 * values[:len(got)]), at
    got = mass.numpy(span, CELLS - span)
    assert (np.abs(got - 0.5 * old[-1] - want) <= near + 2.0 ** -23 * (old[-1] + want)).all()
    assert (mass.numpy(2, CELLS) == 7).all()
    mass.free()
