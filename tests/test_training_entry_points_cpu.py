"""What the C entry points of group norm, linear cross entropy and AdamW refuse on the host: nothing is launched, the addresses are
made up."""
from array import array

import pytest

from warpconvnet_b200 import _native

BASE = 1 << 20   # stands for aligned device memory
INVALID, BOUNDS = -5, -8


def backward(workspace, n=256, c=64, v=40, dtype=_native.WCN_BF16):
    size = _native.query_bytes("wcn_linear_ce_workspace_bytes", n, c, v, dtype, 7)
    return _native.lib().wcn_linear_ce_backward(BASE, c, n, c, BASE, c, v, None, BASE, -100, dtype, BASE, BASE, BASE, BASE, None, BASE, BASE, BASE, dtype,
                                                workspace, size, BASE, None)


@pytest.mark.parametrize("n,c,v", [(256, 64, 40), (256, 64, 1000), (256, 512, 1000)])   # a kernel for each: few classes, many, wide rows
@pytest.mark.parametrize("dtype", [_native.WCN_F32, _native.WCN_F16, _native.WCN_BF16])
def test_workspace_of_the_cross_entropys_gradients_starts_on_32_bytes(n, c, v, dtype):
    """Sums go there in pieces of 32 bytes."""
    for off in (4, 8, 16, 48):
        assert backward(BASE + off, n, c, v, dtype) == INVALID


def step(sizes, slots, length):
    count = len(sizes)
    at, sizes, slots = array("q", [BASE] * count), array("q", sizes), array("q", slots)
    address = lambda a: a.buffer_info()[0]   # noqa: E731
    return _native.lib().wcn_adamw_step(address(at), address(at), address(sizes), address(slots), None, count, 0, 0, BASE, None, BASE, None, length, BASE, count,
                                        0, 0, 0, 0, 0, None, None, None, BASE, None)


@pytest.mark.parametrize("slot", [512, 1 << 40, (1 << 63) - 512, (1 << 63) - 256])
def test_moments_beyond_their_end_are_refused(slot):
    """Also where a slot and a size come to more than 2^63."""
    assert step([300], [slot], 512) == BOUNDS
    assert step([5, 300], [0, slot], 512) == BOUNDS
    assert step([(1 << 63) - 1], [0], 512) == BOUNDS


@pytest.mark.parametrize("dtype,size", [(_native.WCN_F32, 4), (_native.WCN_BF16, 2)])
@pytest.mark.parametrize("n", [1, 130, 3000])
def test_the_logits_gradient_has_pieces_of_512_mb_at_most(dtype, size, n):
    """Whatever the classes are: with it a piece's gradients of the weights in fp32, for up to 23 divisions of 3000 rows."""
    for v in (70_000, 4_300_000, 40_000_000):
        piece = min(v, max(1024, (512 << 20) // (size * n) + 256))
        parts = -(-n // 128)
        assert _native.query_bytes("wcn_linear_ce_workspace_bytes", n, 8, v, dtype, 2) <= (512 << 20) + parts * piece * 16 * 4 + 4 * 16 * v + (1 << 20)
