"""CPU checks of the layouts that the paged-cache operators write through: rows that share
memory are refused before a launch, whatever pair of axes makes them meet."""

import pytest

from umic_b200 import _lib

F = 4096  # never dereferenced: the check under test fails first


def _input(qo=(512, 128), ko=(256, 128), pages=None, num=8, page=16, d=128):
    """Four query and two KV heads, four tokens."""
    sp, sh, ss = pages or (0, 0, 0)
    kp = F if pages else 0
    args = _lib.pack_mrope_args(
        F, F, F, F, 0 if pages else F, 0, 0, 0, 0, kp, kp, 0, 0, F, 512, d, 256, d, 256, d, *qo,
        *ko, 0, 0, sp, sh, ss, num, page, 4, 4, 2, d, 0, 4, 0, 1, 0, 0, 0, 0, 0, 1e-6, 1e-6, 1.0)
    return _lib.lib().umic_qk_norm_mrope_kv(args, None)


@pytest.mark.parametrize("kw", [
    dict(qo=(128, 128)),             # row (t, h + 1) is row (t + 1, h)
    dict(qo=(384, 128)),             # the last head is the next token's first
    dict(qo=(128, 384)),             # heads outside, four tokens of 128 do not fit 384
    dict(ko=(128, 128)),
    dict(ko=(128, 256)),
    dict(ko=(248, 128)),
    dict(pages=(8192, 128, 128)),    # a token of one head is the next head's
    dict(pages=(8192, 1920, 128)),   # 16 tokens do not fit a head
    dict(pages=(2048, 2048, 128)),   # a page's second head is the next page
    dict(pages=(128, 2048, 128)),
    dict(pages=(8192, 128, 248)),    # heads inside tokens, two of them do not fit
    dict(pages=(4088, 2048, 128)),
    dict(pages=(1 << 62, 1 << 62, 128))])  # spans past 64 bits do not wrap
def test_input_rows_that_meet_are_refused(kw):
    assert _input(**kw) == 1
    assert "overlap" in _lib.last_message()


def _attend(out, batch=3, hq=4):
    args = _lib.pack_paged_attention_args(
        F, F, F, 0, 0, F, F, F, 0, F, 512, 128, 4096, 2048, 128, 8, 16, 4, 4, *out, batch, 1 << 30,
        hq, 2, 128, 0, 0.1)
    return _lib.lib().umic_paged_attention(args, None)


@pytest.mark.parametrize("out", [(128, 128), (384, 128), (128, 256), (504, 128), (136, 128)])
def test_attention_rows_that_meet_are_refused(out):
    assert _attend(out) == 1
    assert "overlap" in _lib.last_message()
