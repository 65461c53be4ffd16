"""Which kernels the paged attention's tests run: no GPU needed."""
import pytest

from tensor_fusion_amd.ops import paged

pytestmark = pytest.mark.usefixtures("native_built")


def dispatch(seqs, heads, Hk, D, page, quantized, extra_cols=1):
    """(workers, waves, join, splits) for a batch as the tests make it."""

    cols = max(-(-kv // page) for _, kv in seqs) + extra_cols
    return paged._ext().dispatch(sum(n for n, _ in seqs), len(seqs),
                                 heads // Hk, Hk, D, cols * page, quantized)


@pytest.mark.parametrize("quantized", [False, True])
def test_keys_are_split_where_tests_say_so(quantized):
    """In tests/test_gpu_paged.py."""

    # values that are not finite, in keys that are split
    workers, _, join, splits = dispatch([(3, 6000), (2, 900)], 4, 2, 64, 16,
                                        quantized)
    assert workers and join and splits == 1
    assert dispatch([(60, 4000), (70, 2000)], 4, 2, 64, 16,
                    quantized)[::3] == (0, 16)
    # scales of steps
    for seqs, heads in (([(1, 9000)], 8), ([(2, 9000)], 64)):
        workers, _, join, splits = dispatch(seqs, heads, 4, 128, 64,
                                            quantized)
        assert (workers and join) if seqs[0][0] == 1 else splits > 1
    # captured calls that join
    assert paged._ext().dispatch(2, 2, 4, 4, 128, 8192, quantized)[2] == 1
    assert paged._ext().dispatch(80, 2, 4, 4, 128, 8192, quantized)[3] > 1


def test_plan_is_the_dispatch_of_16_bits():
    ext = paged._ext()
    for sizes in ((1, 1, 1, 1, 128, 0), (64, 64, 8, 8, 128, 8192),
                  (8192, 1, 4, 8, 128, 8192), (40, 1, 4, 8, 64, 700)):
        workers, _, join, splits = ext.dispatch(*sizes, False)
        assert ext.plan(*sizes) == (workers, join, splits)
    with pytest.raises(ValueError, match="arguments"):
        ext.dispatch(1, 1, 1, 1, 128, 0)
    with pytest.raises(ValueError, match="no plan"):
        ext.dispatch(0, 1, 1, 1, 128, 0, True)


def test_waves_and_items():
    """Whole items of an 8-bit cache: 8 waves up to an item for each unit, 4
    past that; shared ones go by what there is."""

    one = [(1, 500)]
    for D in (64, 128):
        assert dispatch(one * 20, 32, 8, D, 32, True)[1:] == (8, 0, 1)
        assert dispatch(one * 40, 32, 8, D, 32, True)[1:] == (4, 0, 1)
        assert dispatch(one * 20, 32, 8, D, 32, False)[1:] == (4, 0, 1)
        assert dispatch([(1, 9000)] * 20, 32, 8, D, 32, True) == (256, 8, 1, 1)
