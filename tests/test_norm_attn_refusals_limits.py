"""CPU: calls of group_norm_act / cross_attn beyond the sizes that the kernels' indexes hold, or with written memory on an operand that is
read beside the rows.  Refused before any HIP call."""
import pytest

from tests.test_norm_attn_refusals import GN_APART, GNB_APART, P, gn, gnb, refused


@pytest.mark.parametrize("n", [1 << 30, (1 << 31) - 1000, (1 << 31) - 1])
def test_group_norm_act_refuses_rows_past_its_indexes(n):
    """A thread steps up to 4 x 512 rows past its last one before it compares: in 32 bits that wraps near 2^31 rows an image."""
    far = dict(B=1, n=n, C=1, G=1, ldx=1, nb=1 << 40)
    refused(gn(**dict(GN_APART, ldo=1, x=P, out=P << 24, ws=P << 26, **far)), "group_norm_act", "shape")
    refused(gnb(**dict(GNB_APART, ldy=1, ldd=1, x=P << 22, dy=P << 23, dx=P << 24, ws=P << 26, **far)), "group_norm_act_backward", "shape")
