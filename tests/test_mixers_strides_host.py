"""Strides of rows of heads that no memory has are refused before a device is
touched, also where a row's length in 64 bits would wrap."""
import pytest

from test_mixers_host import heads


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("sizes,strides", [
    ((5, 1024, 64), (64, 1 << 54, 1)),           # 1023 * 2^54 wraps to below 0
    ((5, 5, 64), (64, 1 << 62, 1)),              # 4 * 2^62 wraps to 0
    ((1, 5, 64), (64, 1 << 61, 1)), ((5, 2, 64), (1 << 61, 64, 1)),
    ((1 << 23, 1, 64), (1 << 45, 64, 1)), ((5, 2, 64), (1 << 62, (1 << 62) - 64, 1))])
def test_strides_without_memory(q8, bf16, sizes, strides):
    assert heads(q8, bf16, sizes=sizes, strides=strides) == q8.DECLINED


@pytest.mark.parametrize("bf16", [False, True])
def test_wide_strides(q8, bf16):
    assert heads(q8, bf16, sizes=(2, 2, 64), strides=(1 << 36, 1 << 30, 1)) == q8.OK
    assert heads(q8, bf16, sizes=(2, 1, 64), strides=(1 << 36, -5, 1)) == q8.OK  # one head: no stride
