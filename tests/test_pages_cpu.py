"""Refusals of the paged cache's operators, on the host (no GPU): the wrappers' and the C entries'."""

import numpy as np
import pytest
import torch

from iron_b200 import _lib
from iron_b200 import kernels as K
from tests import pages_ref as R

I32, BF16, F8 = torch.int32, torch.bfloat16, torch.float8_e4m3fn


def _step(**over):
    a = dict(tables=torch.zeros((3, 4), dtype=I32), lengths=torch.zeros(3, dtype=I32), new_tokens=torch.ones(3, dtype=I32),
             pages=torch.arange(12, dtype=I32), ring=torch.tensor([0, 12, 0, 0], dtype=I32), page_size=16, rows=3)
    a.update(over)
    return K.page_step(**a)


@pytest.mark.parametrize("over, error", [
    (dict(), RuntimeError),                                          # CPU tensors: no fallback
    (dict(lengths=torch.zeros(4, dtype=I32)), ValueError),
    (dict(new_tokens=torch.zeros((3, 1), dtype=I32)), ValueError),
    (dict(tables=torch.zeros(12, dtype=I32)), ValueError),
    (dict(ring=torch.zeros(3, dtype=I32)), ValueError),
    (dict(rows=-1), ValueError),
    (dict(slots=torch.zeros(4, dtype=I32)), ValueError),
    (dict(row_start=torch.zeros(3, dtype=I32)), ValueError),
    (dict(lengths=torch.zeros(3, dtype=torch.int64)), TypeError),
    (dict(pages=torch.arange(12)), TypeError),
])
def test_page_step_refuses(over, error):
    with pytest.raises(error):
        _step(**over)


def _write(H=4, G=2, D=64, rows=3, **over):
    a = dict(qkv=torch.zeros((rows, (H + 2 * G) * D), dtype=BF16), angles=torch.zeros((8, D), dtype=BF16),
             q_out=torch.zeros((rows, H, D), dtype=BF16), pool=torch.zeros((5, G, 2, 16, D), dtype=F8),
             scales=torch.ones((5, G, 2)), slots=torch.zeros(rows, dtype=I32), positions=torch.zeros(rows, dtype=I32))
    a.update(over)
    return K.rope_kv_pages(**a, H=H, G=G, D=D)


@pytest.mark.parametrize("over, error", [
    (dict(), RuntimeError),
    (dict(pool=torch.zeros((5, 2, 2, 16, 64), dtype=torch.uint8)), TypeError),
    (dict(pool=torch.zeros((5, 2, 16, 64), dtype=F8)), ValueError),
    (dict(pool=torch.zeros((5, 3, 2, 16, 64), dtype=F8), scales=torch.ones((5, 3, 2))), ValueError),
    (dict(scales=torch.ones((5, 2))), ValueError),
    (dict(scales=torch.ones((5, 2, 2), dtype=torch.float64)), TypeError),
    (dict(qkv=torch.zeros((3, 512))), TypeError),
    (dict(qkv=torch.zeros((3, 448), dtype=BF16)), ValueError),
    (dict(qkv=torch.zeros((512, 3), dtype=BF16).t()), ValueError),
    (dict(angles=torch.zeros((8, 32), dtype=BF16)), ValueError),
    (dict(q_out=torch.zeros((2, 4, 64), dtype=BF16)), ValueError),
    (dict(slots=torch.zeros(2, dtype=I32)), ValueError),
    (dict(slots=torch.zeros(3, dtype=torch.int64)), TypeError),
])
def test_rope_kv_pages_refuses(over, error):
    with pytest.raises(error):
        _write(**over)


def _attend(prompt, **over):
    a = dict(Q=torch.zeros((3, 4, 64), dtype=BF16), pool=torch.zeros((5, 2, 2, 16, 64), dtype=F8),
             scales=torch.ones((5, 2, 2)), tables=torch.zeros((3, 2), dtype=I32), lengths=torch.ones(3, dtype=I32))
    if prompt:
        a["row_start"] = torch.arange(4, dtype=I32)
    a["workspace"] = torch.zeros(8, dtype=torch.uint8)
    a.update(over)
    return (K.mha_prefill_pages if prompt else K.mha_decode_pages)(**a)


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("over, error", [
    (dict(), RuntimeError),
    (dict(Q=torch.zeros((3, 4, 64))), TypeError),
    (dict(Q=torch.zeros((3, 3, 64), dtype=BF16)), ValueError),
    (dict(Q=torch.zeros((3, 4, 128), dtype=BF16)), ValueError),
    (dict(Q=torch.zeros((3, 256), dtype=BF16)), ValueError),
    (dict(out=torch.zeros((3, 4, 32), dtype=BF16)), ValueError),
    (dict(tables=torch.zeros((4, 2), dtype=I32)), ValueError),
    (dict(tables=torch.zeros((3, 2), dtype=torch.int64)), TypeError),
    (dict(lengths=torch.ones(3)), TypeError),
])
def test_attention_refuses(prompt, over, error):
    with pytest.raises(error):
        _attend(prompt, **over)


def test_decode_takes_one_query_a_request_and_prompts_their_row_starts():
    with pytest.raises(ValueError):
        _attend(False, Q=torch.zeros((2, 4, 64), dtype=BF16))
    with pytest.raises(ValueError):
        _attend(True, row_start=torch.arange(3, dtype=I32))
    with pytest.raises(ValueError):
        _attend(True, causal=False, window=4)
    with pytest.raises(TypeError):
        _attend(True, row_start=torch.arange(4))


def test_the_c_entries_refuse_before_any_launch():
    lib = _lib.load()
    a, shape, align, unsup, small = 16, -1, -2, -4, -5      # `a`: an address that is never followed
    step = lambda B=1, width=1, P=4, page=16, rows=1, ring=a: lib.iron_page_step(  # noqa: E731
        a, width, a, a, B, a, P, ring, page, rows, a, a, a, a, a, None)
    assert step(B=-1) == step(B=lib.iron_page_step_max_requests() + 1) == step(width=0) == step(P=0) == shape
    assert step(page=8) == step(page=48) == step(page=512) == step(rows=-1) == step(ring=None) == shape
    assert step(P=1 << 27, page=16) == shape                # slots past 2^31
    write = lambda H=4, G=2, D=64, page=16, rows=2, pitch=512, q=a, P=4: lib.iron_rope_kv_pages_e4m3(  # noqa: E731
        q, pitch, a, a, a, a, P, page, a, a, rows, H, G, D, 8, None)
    assert write(D=96) == write(page=24) == write(pitch=504) == write(pitch=516) == write(H=0) == write(P=0) == shape
    assert write(q=None) == shape and write(q=8) == align and write(rows=0, q=None) == 0

    def attend(H=4, G=2, D=64, B=2, rows=2, page=16, causal=1, window=-1, scale=1.0, q=a, starts=a, nbytes=1 << 40):
        return lib.iron_mha_prefill_pages_bf16(q, a, a, 4, page, a, 1, a, starts, B, rows, H, G, D, causal, window, scale,
                                               a, nbytes, a, None, None)

    assert attend(H=5) == attend(D=80) == attend(page=17) == attend(scale=0.0) == attend(scale=float("nan")) == shape
    assert attend(q=None) == attend(starts=None) == attend(rows=-1) == shape
    assert attend(q=8) == align and attend(causal=0, window=3) == unsup and attend(nbytes=100) == small
    wide = lambda width, P: lib.iron_mha_prefill_pages_bf16(a, a, a, P, 16, a, width, a, a, 2, 2, 4, 2, 64, 1, -1, 1.0,  # noqa: E731
                                                            a, 1 << 40, a, None, None)
    assert wide(1 << 27, 4) == wide((1 << 27) - 1, 4) == wide(1, 1 << 27) == shape       # indices past 2^31
    assert attend(B=0, q=None) == attend(rows=0, q=None) == 0
    assert lib.iron_mha_decode_pages_bf16(a, a, a, 4, 16, a, 1, a, 2, 6, 4, 64, -1, 1.0, a, 1 << 40, a, None, None) == shape
    assert lib.iron_mha_pages_workspace_bytes(96, 0) == 0 < lib.iron_mha_pages_workspace_bytes(64, 0) < lib.iron_mha_pages_workspace_bytes(64, 1)


def test_the_plain_step_hands_pages_on_in_order():
    """The restatement itself, on a case worked by hand: pages of 2, three free in a ring of 6."""
    got = R.page_step(np.array([[4, -1, -1], [5, 0, -1], [-1, -1, -1]]), [1, 4, 0], [2, -1, 3], np.array([9, 9, 1, 2, 3, 9]),
                      [2, 3, 0, 0], 2, 6)
    assert got["tables"].tolist() == [[4, 1, -1], [5, 0, -1], [2, 3, -1]]
    assert got["slots"].tolist() == [9, 2, 4, 5, 6, -1] and got["positions"].tolist() == [1, 2, 0, 1, 2, 0]
    assert got["lengths"].tolist() == [3, 0, 3] and got["row_start"].tolist() == [0, 2, 2, 5]
    assert got["pages"].tolist() == [0, 9, 1, 2, 3, 5] and got["ring"].tolist() == [5, 2, 0, 5]


def test_the_plain_codes_are_torchs():
    x = np.linspace(-448, 448, 20011)
    want = torch.from_numpy(x).float().to(F8).double().numpy()
    assert np.array_equal(R.e4m3(x.astype(np.float32).astype(np.float64)), want)
    assert [R.scale_of(np.array([v])) for v in (448.0, 449.0, 0.0, 1.75, 1.76)] == [1, 2, 2.0 ** -60, 2.0 ** -8, 2.0 ** -7]


@pytest.mark.parametrize("page", [16, 64, 256])
def test_page_step_refuses_tables_whose_tokens_pass_32_bits(page):
    """Positions are 32-bit: a table wide enough for more tokens is refused before any launch."""
    lib, a, wide = _lib.load(), 16, (1 << 31) // page
    step = lambda width: lib.iron_page_step(a, width, a, a, 1, a, 4, a, page, 1, a, a, a, a, a, None)  # noqa: E731
    assert step(wide) == step((1 << 31) - 1) == -1


def test_without_a_device_there_is_no_status_word():
    if not torch.cuda.is_available():
        assert _lib.load().iron_mha_pages_status_word() is None


@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("status, error", [
    (torch.zeros(1), TypeError), (torch.zeros(1, dtype=torch.uint8), TypeError), (torch.zeros(0, dtype=I32), ValueError),
    (torch.zeros(1, dtype=I32), RuntimeError),                       # a word that the device cannot write
])
def test_a_status_word_is_one_int32_of_the_device(prompt, status, error):
    with pytest.raises(error):
        _attend(prompt, status=status)
