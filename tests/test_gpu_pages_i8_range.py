"""Attention of packed prompts over an 8-bit cache whose values' scales lie far apart, or near the ends of f32's range: each
query's result is right for what it sees, whatever the blocks that it does not see hold."""
import numpy as np
import pytest

from test_gpu_pages_i8 import prompt_case

pytestmark = pytest.mark.gpu

F32 = np.float32


def finite_case(ctx, nnhip, **case):
    """prompt_case, whose bound a NaN would not show in, of finite results alone."""
    assert np.isfinite(prompt_case(ctx, nnhip, **case)).all()


def scaled(c, b, first, count, power):
    """The values' scales of sequence b's blocks first .. first + count - 1 times 2^power (blocks of 16 positions)."""
    per = c.page // c.block
    for i in range(first, first + count):
        at = (c.table[b, i // per], slice(None), i % per)
        c.scales["v"][at] = np.ldexp(c.scales["v"][at], power).astype(F32)


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("dk,H,Hkv", [(64, 1, 1), (128, 8, 1), (64, 4, 2)])
@pytest.mark.parametrize("first,power", [(1, 150), (2, 150), (4, 160), (9, 155), (3, 100), (5, -150), (2, -110)])
def test_blocks_behind(ctx, nnhip, dk, H, Hkv, cap, first, power):
    """From block `first` on values are 2^power of those before: queries of the same 32, tile or work-group as those that see them."""
    def edit(c, q):
        scaled(c, 0, 0, 20, -power // 2)
        scaled(c, 0, first, 20 - first, power)

    finite_case(ctx, nnhip, lens=[320], pos0=[0], H=H, Hkv=Hkv, dk=dk, page=32, block=16, cap=cap, slopes=cap > 0, stride=7, edit=edit)


@pytest.mark.parametrize("power", [150, -150])
def test_blocks_behind_few_queries(ctx, nnhip, power):
    """The same where waves share the keys, and where spans share the item."""
    def edit(c, q):
        for b, n in ((0, 3), (1, 19)):
            scaled(c, b, 0, n, -power // 2)
        scaled(c, 0, 2, 1, power)   # positions 32 .. 44 of queries 20 .. 44
        scaled(c, 1, 18, 1, power)  # 288 .. 303 of queries 270 .. 299

    for H, Hkv in ((4, 1), (2, 2)):
        finite_case(ctx, nnhip, lens=[25, 30], pos0=[20, 270], H=H, Hkv=Hkv, dk=128, page=32, block=16, edit=edit)


@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_alternating_blocks(ctx, nnhip, cap):
    """Scales that go up and down by 2^100 and more along a sequence."""
    powers = (0, -70, 70, 60, -60, -75, 75, 10, 0, -10, 74, -74)

    def edit(c, q):
        for b in range(2):
            for i in range(28 if b else 19):
                scaled(c, b, i, 1, powers[(i + 5 * b) % 12])

    finite_case(ctx, nnhip, lens=[300, 40], pos0=[0, 400], H=4, Hkv=1, dk=128, page=32, block=16, cap=cap, slopes=cap > 0, stride=5,
                edit=edit)


@pytest.mark.parametrize("power", [112, 118, -80])
@pytest.mark.parametrize("lens,pos0", [([300], [0]), ([256, 100], [700, 0]), ([10], [2000]), ([1, 1], [700, 40]), ([40], [1200])])
def test_ends_of_the_range(ctx, nnhip, lens, pos0, power):
    """Values about 2^115 over hundreds of keys, by one work-group, by waves that share keys and by spans that share items: their
    weighted mean is as large as they are. And small ones."""
    def edit(c, q):
        for b in range(len(lens)):
            n = -(-(lens[b] + pos0[b]) // 16)
            most = max(float(np.max(c.scales["v"][c.table[b, i // 2], :, i % 2])) for i in range(n))
            scaled(c, b, 0, n, power - int(np.ceil(np.log2(most))) - 1)  # scales of up to 2^(power - 1), values below 2^(power + 6)

    for H, Hkv, dk in ((4, 4, 64), (8, 1, 128)):
        finite_case(ctx, nnhip, lens=lens, pos0=pos0, H=H, Hkv=Hkv, dk=dk, page=32, block=16, stride=9, edit=edit)


@pytest.mark.parametrize("cap,slopes", [(0.0, False), (20.0, True), (0.0, True)])
@pytest.mark.parametrize("lens,pos0", [([70], [0]), ([9], [300]), ([200], [200])])
def test_zero_keys_of_large_scales(ctx, nnhip, lens, pos0, cap, slopes):
    """Codes of 0 under scales that pass f32's range times the query's size stand for 0, and scores are 0."""
    def edit(c, q):
        c.codes["k"][:] = 0
        c.scales["k"][:] = F32(2.0 ** 100)
        q *= F32(2.0 ** 90)

    finite_case(ctx, nnhip, lens=lens, pos0=pos0, H=4, Hkv=1, dk=128, page=32, block=16, cap=cap, slopes=slopes, rope=False, stride=7, edit=edit)
