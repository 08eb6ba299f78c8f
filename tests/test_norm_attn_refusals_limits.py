"""CPU: calls of group_norm_act / cross_attn beyond the sizes that the kernels' indexes hold, or with written memory on an operand that is
read beside the rows.  Refused before any HIP call."""
import pytest
import torch

from underwater_image_restoration_amd import ops
from tests.test_norm_attn_refusals import GN_APART, GNB_APART, P, SPLIT, ca, cab, gn, gnb, refused


@pytest.mark.parametrize("n", [1 << 30, (1 << 31) - 1000, (1 << 31) - 1])
def test_group_norm_act_refuses_rows_past_its_indexes(n):
    """A thread steps up to 4 x 512 rows past its last one before it compares: in 32 bits that wraps near 2^31 rows an image."""
    far = dict(B=1, n=n, C=1, G=1, ldx=1, nb=1 << 40)
    refused(gn(**dict(GN_APART, ldo=1, x=P, out=P << 24, ws=P << 26, **far)), "group_norm_act", "shape")
    refused(gnb(**dict(GNB_APART, ldy=1, ldd=1, x=P << 22, dy=P << 23, dx=P << 24, ws=P << 26, **far)), "group_norm_act_backward", "shape")


# key_lens and key_mask are read while outputs, lse and the workspace are written
@pytest.mark.parametrize("kw,words", [
    (dict(lens=P << 4), ("out", "key_lens")), (dict(mask=(P << 4) + 100, ldm=20), ("out", "key_mask")), (dict(lse=P << 8, lens=(P << 8) + 8), ("lse", "key_lens")),
    (dict(lse=P << 8, mask=(P << 8) - 39, ldm=20), ("lse", "key_mask")), (dict(SPLIT, lens=(P << 9) + 4), ("workspace", "key_lens")),
    (dict(SPLIT, mask=(P << 9) - 16, ldm=8192), ("workspace", "key_mask"))])
def test_cross_attn_refuses_lengths_and_masks_in_written_memory(kw, words):
    refused(ca(**kw), "cross_attn", "overlaps", *words)


@pytest.mark.parametrize("kw,words", [
    (dict(lens=P << 5), ("dq", "key_lens")), (dict(mask=(P << 6) + 2, ldm=20), ("dk", "key_mask")), (dict(lens=(P << 7) + 4), ("dv", "key_lens")),
    (dict(lens=P << 8), ("workspace", "key_lens")), (dict(mask=P << 8, ldm=64), ("workspace", "key_mask"))])
def test_cross_attn_backward_refuses_lengths_and_masks_in_written_memory(kw, words):
    refused(cab(**dict(dict(lse=P << 10), **kw)), "cross_attn_backward", "overlaps", *words)


def test_host_operands_are_named_in_the_error():
    q, k = torch.zeros(10, 64), torch.zeros(20, 64)
    with pytest.raises(ValueError, match="operand on cpu: every operand of an op is a tensor on the current HIP device"):
        ops.cross_attn(q, k, k, 2, 5, 10, 2, 2, 32, 0.5, torch.zeros(10, 64), None)
    with pytest.raises(ValueError, match="operand on meta: every operand"):
        ops._stream(torch.device("meta"))
