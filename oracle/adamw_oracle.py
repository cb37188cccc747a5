"""TEST INFRASTRUCTURE ONLY.  One AdamW step in float64 numpy, with the roundings of its stored forms: bf16 parameters and e4m3
moments (m to nearest, sqrt(v) stochastically), and the random bits that decide them.  The reference has no trainer.  Only tests may
import this module."""
import numpy as np

BLOCK = 256


def stir(x):
    x = np.asarray(x, np.uint64) & 0xFFFFFFFF
    x ^= x >> np.uint64(16)
    x = (x * np.uint64(0x6A09E667)) & np.uint64(0xFFFFFFFF)
    x ^= x >> np.uint64(15)
    x = (x * np.uint64(0xBB67AE85)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def random_bits(n, index, step, seed):
    key = stir(np.uint64(index) ^ stir(np.uint64(step) ^ stir(np.uint64(seed))))
    return stir(np.arange(n, dtype=np.uint64) ^ key)


def spacing(x, digits, least):
    """Distance, at |x|, of the values with `digits` bits behind the leading one and 2^least as the smallest normal number."""
    return np.exp2(np.maximum(np.frexp(np.abs(x))[1] - 1, least) - float(digits))


def up_or_down(x, grid, u):
    """x onto the grid: down, or up where u in [0, 1) and the part above the lower neighbour add up to a step."""
    return np.copysign(np.floor(np.abs(x) / grid + u) * grid, x)


def values_of(codes, scales):
    return codes * np.repeat(scales, BLOCK)[:len(codes)]


def update(p, g, m, v, step, lr, b1, b2, eps, decay):
    """(p, m, v) in float64."""
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return p * (1 - lr * decay) - lr / (1 - b1 ** step) * m / (np.sqrt(v / (1 - b2 ** step)) + eps), m, v


def bf16_stochastic(x, random):
    return up_or_down(x, spacing(x, 7, -126), (random & np.uint64(0xFFFF)).astype(np.float64) / 65536)


def block_scales(x):
    pad = np.concatenate((np.abs(x), np.zeros(-len(x) % BLOCK))).reshape(-1, BLOCK)
    return pad.max(1) / 448


def e4m3_nearest(q):
    grid = spacing(q, 3, -6)
    return np.rint(q / grid) * grid


def e4m3_stochastic(q, random):
    """q >= 0; never to zero from above it."""
    r = up_or_down(q, spacing(q, 3, -6), (random >> np.uint64(16)).astype(np.float64) / 65536)
    return np.where(q > 0, np.clip(r, 2.0 ** -9, 448.0), 0.0)
