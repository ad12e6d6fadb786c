"""Host arithmetic of the cache: rows of outputs that lie on one another are found, against all pairs of rows, and refused; how far quotients are from the middles of codes."""
import ctypes
import itertools
import random

import pytest

from pi05_megakernel_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def numbers(v):
    return (ctypes.c_longlong * len(v))(*v)


def meet(lib, size, stride, width, other=None, distance=0):
    b = (None, None) if other is None else (numbers(other[0]), numbers(other[1]))
    return lib.pi05_rows_meet(len(size), numbers(size), numbers(stride), *b, distance, width)


def places(size, stride, at=0):
    return [at + sum(i * s for i, s in zip(index, stride)) for index in itertools.product(*(range(n) for n in size))]


def test_against_all_pairs(lib):
    rng = random.Random(5)
    found = [0, 0, 0, 0]
    for _ in range(6000):
        width = 8 * rng.choice((1, 2, 8))
        tensor = lambda: ([rng.randint(0 if rng.random() < 0.05 else 1, 4) for _ in range(4)],
                          [8 * rng.choice((0, 1, 2, 3, 5, 8, 9, 16, 17, 24, 33, 64, 100)) * rng.choice((1, 1, 1, -1)) for _ in range(4)])
        a, b = tensor(), tensor()
        rows = sorted(places(*a))
        same = any(y - x < width for x, y in zip(rows, rows[1:]))
        assert meet(lib, *a, width) == same, (a, width)
        distance = 8 * rng.randint(-80, 80)
        if rng.random() < 0.4:
            b = a
        both = any(abs(x - y) < width for x in rows for y in places(*b, distance))
        assert meet(lib, *a, width, b, distance) == both, (a, b, width, distance)
        found[same] += 1
        found[2 + both] += 1
    assert min(found) > 500                                               # (both answers, both ways)


def test_usual_layouts_at_any_size(lib):
    """Dense, transposed, cut out of wider tensors, interleaved with one another: none meet; one element more and they do."""
    big = (1 << 20, 18, 1 << 20, 8)
    dense = (18 << 31, 1 << 31, 2048, 256)
    assert meet(lib, big, dense, 256) == 0
    assert meet(lib, big, (1 << 31, 1 << 51, 2048, 256), 256) == 0        # layers outside
    assert meet(lib, (6, 1, 5, 1), (12800, 0, 2560, 0), 256) == 0         # a slice of a projection's output
    assert meet(lib, big, (18 << 31, 1 << 31, 2040, 256), 256) == 1       # the last head over the next token's first
    assert meet(lib, (4, 4, 4, 4), (8, 32, 128, 512), 8) == 0 and meet(lib, (4, 4, 4, 4), (8, 32, 128, 512), 9) == 1
    # keys and values of a token side by side, of a tensor twice as wide
    wide = (36 << 31, 2 << 31, 4096, 256)
    assert meet(lib, big, wide, 256, (big, wide), 2048) == 0 and meet(lib, big, wide, 256, (big, wide), -2048) == 0
    assert meet(lib, big, wide, 256, (big, wide), 2047) == 1 and meet(lib, big, wide, 256, (big, wide), 0) == 1
    assert meet(lib, big, dense, 256, (big, dense), 18 << 51) == 0 and meet(lib, big, dense, 256, (big, dense), (18 << 51) - 2048) == 1
    # queries [tokens][sequences][q | k | v], outputs dense beside them, and queries that are expanded
    assert meet(lib, (64, 8, 8), (2560, 163840, 256), 256, ((64, 8, 8), (16384, 2048, 256)), 1310720) == 0
    assert meet(lib, (64, 8, 8), (0, 2048, 256), 256, ((64, 8, 8), (16384, 2048, 256)), 16384) == 0
    assert meet(lib, (64, 8, 8), (0, 2048, 256), 256, ((64, 8, 8), (16384, 2048, 256)), 16128) == 1
    assert meet(lib, (0, 8), (0, 0), 64) == 0 and meet(lib, (1, 1), (0, 0), 64) == 0


def test_entry_points_refuse(lib):
    """No pointer is followed: refused before a device is asked for (and without a GPU what is not refused ends there)."""
    from test_cache_host import cache, call, rows
    fine = (_lib.ERR_NO_DEVICE,)
    for change in (dict(v=0x60000), dict(v=0x60010), dict(head_stride=120), dict(token_stride=0), dict(batch_stride=0), dict(layer_stride=4096),
                   dict(token_stride=128), dict(batch_stride=8)):
        assert lib.pi05_cache_read(0, cache(), rows(**change), None) == _lib.ERR_ARGUMENT, change
    for change in (dict(out_batch_stride=0), dict(out_head_stride=64), dict(out_batch_stride=1016), dict(out=0x60000), dict(out=0x60010), dict(out=0x60100)):
        assert lib.pi05_shared_attention(0, cache(), call(**change), 0x100000, 1 << 30, None) == _lib.ERR_ARGUMENT, change
    import torch
    if not torch.cuda.is_available():
        for change in (dict(), dict(v=0x60000 + 2 * 8192), dict(batch_stride=2048, layer_stride=4096)):
            assert lib.pi05_cache_read(0, cache(), rows(**change), None) in fine
        # keys and values that are read may lie on one another
        assert lib.pi05_cache_write(0, cache(), rows(v=0x60000, token_stride=0), None) in fine
        for change in (dict(), dict(out=0x60000 + 2 * 2048), dict(q_batch_stride=0), dict(q_head_stride=0)):
            assert lib.pi05_shared_attention(0, cache(), call(**change), 0x100000, 1 << 30, None) in fine


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_quotients_of_codes_are_middles_or_far_from_them(fmt):
    """What the one FP32 quotient of a write rests on: x peak / max|x| of two BF16 numbers is a middle of two codes exactly or at least 2^-16 (int8) and 2^-12.9 (e4m3) of
    itself away from it.  In whole numbers, over all pairs of mantissas and all exponents that codes reach."""
    import numpy as np
    a, x = (v.ravel().astype(np.int64) for v in np.meshgrid(np.arange(128, 256), np.arange(128, 256)))
    if fmt == "int8":
        peak, down, middles = 127, range(0, 10), np.arange(1, 256, 2, dtype=np.int64) << 9          # in units of 2^-10
    else:
        peak, down = 448, range(0, 20)
        values = np.array([m * 2 if e == 0 else (8 + m) << e for e, m in (divmod(c, 8) for c in range(127))], dtype=np.int64)      # of 2^-10
        middles = (values[:-1] + values[1:]) // 2
    nearest = np.inf
    for e in down:
        for i in (0, -1):
            top = peak * x << 10                                          # quotient = top / (a << e), in the middles' units
            at = np.clip(np.searchsorted(middles, top // (a << e)) + i, 0, len(middles) - 1)
            off = np.abs(top - middles[at] * (a << e))
            far = (off > 0) & (x <= a << e)                               # (x is not larger than max|x|)
            nearest = min(nearest, (off[far] / top[far]).min())
    assert nearest >= 2.0 ** (-16 if fmt == "int8" else -12.9), np.log2(nearest)
