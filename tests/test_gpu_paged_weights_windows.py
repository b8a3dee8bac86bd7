"""paged_key_weights of several row tiles by the kernel that goes over the keys for each: the
later ones have only the keys that they see, every key of a row tile in one wave."""
import pytest
import torch

from tests.test_gpu_paged_weights import BF16, F16, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv", [(2, 1), (8, 2), (9, 3), (20, 5), (16, 8), (36, 9), (36, 12), (17, 17)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [1, 33, 64, 200, 1000])
def test_windows_and_heads(gpu, hq, hkv, causal, window):
    g = hq // hkv
    lens = [700, 2000, 65, 9, 33, 1300]
    for n in (33 // g + 1, 96 // g, 128 // g):
        run(gpu, lens, [n] * len(lens), hq, hkv, 64, F16, causal=causal, window=window, uniform=True, decay=0.5,
            name=f"{hq}/{hkv} {n} rows, window {window}")


@pytest.mark.parametrize("d,i8,dtype", [(128, False, BF16), (128, True, F16), (256, False, F16), (64, True, BF16)])
@pytest.mark.parametrize("window", [-1, 50])
def test_more_row_tiles_than_said(gpu, d, i8, dtype, window):
    """A max_seqlen_q below the rows: any number of row tiles, on sequences split over workers."""
    run(gpu, [6000, 900, 300], [70, 300, 300], 8, 2, d, dtype, i8, window=window, max_q=1,
        name=f"said 1, window {window}")


@pytest.mark.parametrize("window", [40, 300])
def test_long_sequences(gpu, window):
    run(gpu, [30000, 20011], [60, 31], 8, 4, 64, BF16, window=window, decay=0.9, spoil=True, name=f"long {window}")
    run(gpu, [30000, 20011], [60, 31], 8, 4, 64, BF16, window=window, causal=False, page=1, name=f"pages of 1 {window}")
