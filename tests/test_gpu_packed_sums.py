"""Row sums of packed attention over many keys of small weight, against their closed form in 64 bits."""

import math

import pytest
import torch

import serving_reference as ref
from reskv_amd import packed_attention

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("bits", [17.4, 20.3, 22.6])
@pytest.mark.parametrize("n", [1 << 16, 1 << 19])
@pytest.mark.parametrize("most", [0, None])
def test_many_keys_far_below_one(device, n, bits, most):
    """One key of value 1 above n - 1 others of value 0 whose weights are 2^-bits of its own: 1 / (1 + (n - 1) 2^-bits),
    with the keys whole (max_keys = 0) and split.

    Roundings: of a weight, 2^-11, and of the result; in fp32, of scores below 2^5 (2^-20 of a weight), and of sums: the
    lanes' 32 weights of a tile, n / 64 tiles one after the other, and a key's value over n / 16 products
    of 16 keys, each at most 2^-24 of the sum that it is added to."""
    q = torch.zeros(1, 1, 128, dtype=torch.float16, device="cuda")
    k, v = (torch.zeros(n, 1, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    q[0, 0, 0], v[0] = 16, 1
    k[0, 0, 0] = bits * math.log(2) * 128 ** 0.5 / 16
    score = 16 * k[0, 0, 0].double().item() * 128 ** -0.5
    want = 1 / (1 + (n - 1) * math.exp(-score))
    bound = want * (2 * ref.H16 + 2.0 ** -19 + (n / 64 + n / 16 + 32) * ref.H32)
    got = packed_attention(q, k, v, i32([0, 1]), i32([0, n]), max_keys=most).double()
    assert (got - want).abs().max().item() <= bound


def test_a_first_key_that_outweighs_a_long_prompt(device):
    """A prompt whose first key has nearly all of every row's weight and a small value, as models leave it: the
    rest, thousands of weights of 2^-22 and less, makes the result."""
    n = 6000
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn(n, 1, 128, generator=g, device="cuda").half()
    k = torch.randn(n, 1, 128, generator=g, device="cuda").half()
    v = torch.randn(n, 1, 128, generator=g, device="cuda").half() + 2
    q[:, 0, 0], k[:, 0, 0] = 12, 0
    k[0], v[0] = 0, 2.0 ** -12
    k[0, 0, 0] = 14.5
    got = packed_attention(q, k, v, i32([0, n]))
    rows = [0, 1, 63, 64, 1000, 3000, n - 1]
    for r in rows:
        w, b = ref.sequence(q[r: r + 1].double().cpu().numpy(), k[: r + 1].double().cpu().numpy(),
                            v[: r + 1].double().cpu().numpy(), r, 128 ** -0.5)
        assert (abs(got[r: r + 1].double().cpu().numpy() - w) <= b).all(), r
