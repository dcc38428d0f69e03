"""Why the moments' codes are rounded stochastically: the codes of _adamw_reference.py over many steps against exact moments."""
import numpy as np

from tests._adamw_reference import decode, encode, moments32, random_bits

B1, B2 = 0.9, 0.999


def _run(n, steps, stochastic):
  """Mean ratio of coded to exact second moments after `steps` steps of Gaussian gradients, scales from 1e-3 to 1e-1 in a block."""
  rng = np.random.default_rng(0)
  sigma = 10.0 ** rng.uniform(-3, -1, n)
  m = v = exact = np.zeros(n)
  for t in range(1, steps + 1):
    g = (sigma * rng.standard_normal(n)).astype(np.float32)
    exact = B2 * exact + (1 - B2) * g.astype(np.float64) ** 2
    m, v = moments32(g, m, v, B1, B2)
    x = random_bits(0, t, 0, n)
    m = decode(*encode(m, 3, (x >> 12) / 2.0 ** 20 if stochastic else np.full(n, 0.5)), 3)
    v = decode(*encode(v, 2, (x & 0x1FFFFF) / 2.0 ** 21 if stochastic else np.full(n, 0.5)), 2)
  return np.mean(v / exact), np.std(np.log2(v / exact))


def test_stochastic_rounding_follows_the_second_moment_and_rounding_to_nearest_does_not():
  """Stochastic: the expectation is the exact moment.  A step moves v by d = (1 - b2) (g^2 - v) off its code, the rounding adds a
  variance of at most |d| times the spacing, v / 4 at most: (1 - b2) (s^2 v + v^2) / 4 in the mean for gradients of variance s^2,
  and with the sum of b2^(2k) over 1 / (1 - b2^2) steps a variance of 0.28 s^4 (its own part in v^2 included): 0.53 of the moment
  an element, 0.53 / sqrt(4096) in their mean, six of which are 0.05.
  Nearest: v rises from a code only where d is half a spacing, v / 16 at least, that is where g^2 >= 63 v: never beyond
  max(g^2) / 63, and no Gaussian out of 4096 * 1000 is beyond 5.5 sigma: 0.48 of the moment."""
  mean, spread = _run(4096, 1000, True)
  assert abs(mean - 1.0) <= 0.05, (mean, spread)
  mean, spread = _run(4096, 1000, False)
  assert mean <= 0.5, (mean, spread)
