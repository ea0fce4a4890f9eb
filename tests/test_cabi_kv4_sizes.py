"""CPU: the attention's workspace size is 0 for sizes that the call refuses, however large."""

import pytest

from esimd_learning_amd import cabi


@pytest.mark.parametrize("T,R,n_q,n_kv,hd,mq,mk", [
    (2 ** 62, 1, 32, 8, 128, 1, 0), (2 ** 62, 2 ** 62, 32, 1, 128, 0, 0), (2 ** 63 - 1, 2 ** 63 - 1, 8, 2, 64, 1, 0),
    (2 ** 31, 1, 32, 8, 128, 1, 0), (2 ** 28, 2 ** 20, 8, 2, 64, 1, 0), (4, 2 ** 26 + 1, 32, 8, 128, 1, 0),
    (4, 1, 8, 2, 64, -1, 0), (4, 1, 8, 2, 64, 1, -1), (4, 1, 2 ** 20, 2 ** 20, 64, 1, 0), (4, 1, 65536, 8, 64, 1, 0),
    (4, 1, 5000, 5000, 64, 1, 0)])
def test_refused_sizes_need_no_workspace(T, R, n_q, n_kv, hd, mq, mk):
    assert cabi.load().cek_kv4_attention_workspace_size(T, R, n_q, n_kv, hd, mq, mk) == 0


def test_the_largest_sizes():
    size = cabi.load().cek_kv4_attention_workspace_size
    assert 0 < size(2 ** 26 - 1, 2 ** 26 - 1, 8, 1, 64, 1, 0) < 2 ** 40     # a row's entry is 16 bytes
    assert size(1, 1, 65535, 1, 256, 1, 0) == 0                              # enough tiles of rows: keys stay whole
