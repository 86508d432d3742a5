"""Host-side checks of the 4-bit KV cache and of sampling, without a device: sizes,
refusals before any launch, and the page layout's bookkeeping."""
import ctypes

import pytest
import torch

from runtimed_b200 import _lib, kv4, sampling
from runtimed_b200.errors import ConfigError, ShapeError


@pytest.mark.parametrize("head_dim,ok", [(32, True), (64, True), (96, True), (128, True), (0, False), (16, False), (80, False),
                                         (160, False), (-32, False)])
def test_page_bytes(head_dim, ok):
    n = ctypes.c_int64(-1)
    rc = _lib.lib().rtd_kv4_page_bytes(head_dim, ctypes.byref(n))
    if ok:
        # 16 tokens, K and V: half a byte a code and a 4-byte header for 32 of them
        want = 16 * 2 * (head_dim // 2 + 4 * (head_dim // 32))
        assert rc == 0 and n.value == want == kv4.page_bytes(head_dim)
    else:
        assert rc == _lib.RTD_ERR_SHAPE and str(head_dim).encode() in _lib.lib().rtd_last_error(None)
        with pytest.raises(ConfigError):
            kv4.page_bytes(head_dim)


def test_null_handles_are_refused():
    L = _lib.lib()
    assert L.rtd_kv4_page_bytes(64, None) == _lib.RTD_ERR_INVALID
    assert L.rtd_kv_plan(None, None, 0, None, None, 1, None, None, 1, None, None, None, None, 0, None) == _lib.RTD_ERR_INVALID
    assert L.rtd_rope_kv4_append(None, None, 1, None, 1, None, 1, 0, 1, 1, 1, 64, 0, None, None, None, None, 1, None,
                                 None) == _lib.RTD_ERR_INVALID
    assert L.rtd_kv4_read(None, None, 1, 1, 64, None, 1, None, None, 0, None) == _lib.RTD_ERR_INVALID
    assert L.rtd_attention_kv4(None, None, 0, 1, 1, 1, 1, 64, 1.0, None, None, 1, None, 1, 1, 1, None, 1, None, 0, 1,
                               None) == _lib.RTD_ERR_INVALID
    assert L.rtd_sample(None, None, 0, 1, 1, 1, None, None, None, None, None, None, None) == _lib.RTD_ERR_INVALID


def test_host_tensors_are_refused():
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros((1, 2, 64))
    pages = torch.zeros((1, 2, 1280), dtype=torch.uint8)
    with pytest.raises(ConfigError):
        kv4.plan(i, i, i[None], i, i)
    with pytest.raises(ConfigError):
        kv4.append(x, x, x, kv4.rope_frequencies(64, 1e4, "cpu"), i, i, pages)
    with pytest.raises(ConfigError):
        kv4.read(pages, i)
    with pytest.raises(ConfigError):
        kv4.attention(x, pages, i[None], torch.zeros(2, dtype=torch.int32), i, 1, 1)
    with pytest.raises(ConfigError):
        sampling.sample(torch.zeros((1, 5)), torch.zeros(1))
    with pytest.raises(ShapeError):
        sampling.sample(torch.zeros(5), torch.zeros(1))


def test_rope_frequencies():
    f = kv4.rope_frequencies(8, 1e6, "cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, 1e6 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8), rtol=1e-14)
    assert kv4.rope_frequencies(0, 1e6, "cpu").numel() == 0
