"""Where the serving operators take scratch, which is where attention over pages divides the keys: both borders from both sides,
without a GPU."""
import pytest

import nnh


def paged(N, rows, most, keys, H, Hkv, D=64):
    return nnh.workspace_size("paged_attention", N, rows, most, keys, H, Hkv, D)


@pytest.mark.parametrize("D", [1, 64, 128])
@pytest.mark.parametrize("N,rows,most,H,Hkv", [(1, 1, 1, 8, 2), (1, 1, 1, 1, 1), (1, 64, 64, 4, 4), (1, 8, 8, 64, 8), (70, 70, 1, 8, 2), (3, 9, 4, 6, 3)])
def test_few_columns_are_divided_from_1024_places(N, rows, most, H, Hkv, D):
    for keys in (0, 1, 16, 512, 1023):
        assert paged(N, rows, most, keys, H, Hkv, D) == 0, keys
    for keys in (1024, 8192):
        assert paged(N, rows, most, keys, H, Hkv, D) > 0, keys


@pytest.mark.parametrize("D", [1, 64, 128])
@pytest.mark.parametrize("rows,H,Hkv", [(65, 4, 4), (9, 64, 8), (33, 2, 1), (1000, 8, 8)])
def test_chunks_are_divided_from_512_places(rows, H, Hkv, D):
    """A sequence of more than 64 columns alone; beside others the single tokens' border is the higher one."""
    for keys in (0, 16, 511):
        assert paged(1, rows, rows, keys, H, Hkv, D) == 0, keys
    for keys in (512, 1023, 1024):
        assert paged(1, rows, rows, keys, H, Hkv, D) > 0, keys
    assert paged(2, rows + 1, rows, 511, H, Hkv, D) == 0 < paged(2, rows + 1, rows, 512, H, Hkv, D) < paged(2, rows + 1, rows, 1024, H, Hkv, D)


def test_many_rows_are_not_divided():
    """Where sequences and heads alone bring eight workgroups of 768, or a chunk's columns 512."""
    assert paged(767, 767, 1, 8192, 32, 8, 128) > 0 == paged(768, 768, 1, 8192, 32, 8, 128)
    assert paged(1, 8191, 8191, 8192, 8, 8) > 0 == paged(1, 8192, 8192, 8192, 8, 8)


@pytest.mark.parametrize("rows", [1, 2, 511, 512, 513, 100000])
def test_sampling_takes_scratch_by_the_vocabulary(rows):
    """With any number of rows, up to that of 512 of them."""
    for code in (nnh.F32, nnh.BF16):
        assert nnh.workspace_size("sample", code, rows, 8192) == 0
        assert nnh.workspace_size("sample", code, rows, 8193) > 0
        assert nnh.workspace_size("sample", code, rows, 8193) <= nnh.workspace_size("sample", code, 512, 8193)


def test_fewer_rows_may_take_more():
    """A workspace for several shapes is sized by asking for each: the largest batch's is not the largest."""
    few, many = (nnh.workspace_size("linear_int8", rows, 4096, 4096) for rows in (1024, 4096))
    assert few > 2 * many > 0
    assert paged(767, 767, 1, 8192, 32, 8, 128) > paged(768, 768, 1, 8192, 32, 8, 128)
