"""sc_gdn_chunk_async over prompts that are longer than a piece of the workspace, by workgroups of 32 columns.  What may differ is
Layer.check's."""
import pytest

from test_gpu_gdn import Layer

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    import sc_ops
    return sc_ops


@pytest.fixture(scope="module")
def plain():
    from oracle import sc_ops
    return sc_ops


# the first has pieces that end inside a sequence, the second sequences that are longer than a piece of 128 chunks
BATCHES = [("f16", 2, 16, [2200, 64, 2111, 3000, 1, 4100, 2000, 2500, 0, 2300, 63, 3333, 2600, 1900, 4000, 3500]), ("f32", 2, 128, [8400, 8700])]


@pytest.mark.parametrize("dtype,kh,vh,lens", BATCHES, ids=["many", "long"])
def test_long_prompts_by_32_columns(sc, ops, plain, cuda, dtype, kh, vh, lens):
    assert len(lens) * vh * 2 >= 512 and sum(-(-n // 64) for n in lens) > 64 * min(len(lens), 8)
    x = Layer(sc, ops, 21, 64, kh, vh, lens, dtype)
    x.build().launch()
    sc.device_sync()
    x.check(plain, heads=[0, vh - 1])
