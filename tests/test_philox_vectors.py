"""The bits of dropout against Philox 4x32-10's published test vectors: a plain form that gives them, and with it the mask that
the other tests expect and the one that the kernels use."""
import pytest
import torch
from test_gpu_dropout import kept

# (counter, key, result): Random123's known answers of ten rounds
VECTORS = [([0] * 4, [0] * 2, [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]),
           ([0xffffffff] * 4, [0xffffffff] * 2, [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]),
           ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0], [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1])]
# (row, chunk, seed, offset); the first is the first vector
PLACES = [(0, 0, 0, 0), (0, 3, 0xa409382213198a2e, 0), (70000, 0, 1, 0x85a308d3243f6a88), (65537, 5, 2 ** 64 - 1, 2 ** 64 - 1)]


def _philox(c, k):
    c, k = list(c), list(k)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [b >> 32 ^ c[1] ^ k[0], b % 2 ** 32, a >> 32 ^ c[3] ^ k[1], a % 2 ** 32]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def _halves(row, chunk, seed, offset):
    words = _philox([chunk, row, offset % 2 ** 32, offset >> 32], [seed % 2 ** 32, seed >> 32])
    return [h for w in words for h in (w & 65535, w >> 16)]


@pytest.mark.parametrize("counter,key,result", VECTORS)
def test_plain_form(counter, key, result):
    assert _philox(counter, key) == result


@pytest.mark.parametrize("row,chunk,seed,offset", PLACES)
def test_expected_mask(row, chunk, seed, offset):
    """A half is kept by its own bound and dropped by the next one."""
    for i, h in enumerate(_halves(row, chunk, seed, offset)):
        at = 8 * chunk + i
        assert kept([row], at + 1, h, seed, offset)[0, at] and not kept([row], at + 1, h + 1, seed, offset)[0, at]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("row,chunk,seed,offset", PLACES)
def test_kernels_mask(row, chunk, seed, offset, dtype):
    from bitsparse_amd.dropout import Dropout, dropout
    from bitsparse_amd.residual import block_join
    x = torch.ones(row + 1, 8 * chunk + 8, device="cuda", dtype=dtype)
    for i, h in enumerate(_halves(row, chunk, seed, offset)):
        for below, stays in ((h, True), (h + 1, False)):
            drop = Dropout(below / 65536, seed, offset)
            assert (dropout(x, drop)[row, 8 * chunk + i].item() != 0) == stays
            assert (block_join(torch.zeros_like(x), x, drop=drop)[row, 8 * chunk + i].item() != 0) == stays
