"""AdamW, the gradient norm and the 8-bit moment codes from their definitions, in numpy: float64 for values, float32
operation by operation where bits are compared (IEEE arithmetic rounds the same everywhere)."""
import numpy as np

U = 2.0 ** -24     # half a unit in the last place of float32, relative
TINY = 2.0 ** -140
C1, C2, C3, C4 = 0x9E3779B1, 0x6A09E667, 0xBB67AE85, 0x3C6EF373
M32 = 0xFFFFFFFF


def adamw64(w, g, m, v, t, lr, b1, b2, eps, wd):
  """One step in float64 and how far a float32 step may be from it: (w, m, v, tol_w, tol_m, tol_v).
  m: four roundings of each addend and one of the sum (constants, product, scaled gradient with its coefficient's four);
  v: twice as many, the gradient enters squared.  w: the quotient's relative error is m's against the sum of its addends'
  magnitudes (12 U), half of v's and the root's, the product's and the sum's roundings (9 + 4 U), the step size's and the
  quotient's (7 U): 32 U; the decayed weight's own roundings 4 U."""
  w, g, m, v = (np.asarray(x, np.float64) for x in (w, g, m, v))
  a, b = b1 * m, (1 - b1) * g
  c, d = b2 * v, (1 - b2) * g * g
  m2, v2 = a + b, c + d
  step = lr / (1 - b1 ** t)
  denom = np.sqrt(v2) / np.sqrt(1 - b2 ** t) + eps
  w2 = w * (1 - lr * wd) - step * m2 / denom
  tol_m = 12 * U * (np.abs(a) + np.abs(b)) + TINY
  tol_v = 18 * U * (c + d) + TINY
  tol_w = 4 * U * np.abs(w) + 32 * U * step * (np.abs(a) + np.abs(b)) / denom + 2 * U * np.abs(w2) + TINY
  return w2, m2, v2, tol_w, tol_m, tol_v


def random_bits(seed, step, tensor, n, first=0):
  k = (seed * C1 + step * C3 + tensor * C4) & M32
  k = ((k ^ (k >> 16)) * C2) & M32
  k = ((k ^ (k >> 15)) * C3) & M32
  k ^= k >> 16
  i = np.arange(first, first + n, dtype=np.uint64)
  x = ((i & M32) * C1 + (i >> np.uint64(32)) * C4 + k) & M32
  x = ((x ^ (x >> 14)) * C2) & M32
  return (x ^ (x >> 14)).astype(np.int64)


def _blocks(x, n):
  out = np.zeros((n + 127) // 128 * 128, x.dtype)
  out[:n] = x
  return out.reshape(-1, 128)


def decode(code, scale_byte, digits):
  """Codes of e4m3 (digits 3) or e5m2 (digits 2) with one scale byte per 128, as float64."""
  bias = 7 if digits == 3 else 15
  c = _blocks(np.asarray(code, np.uint8), len(code)).astype(np.int64)
  e, f = (c & 127) >> digits, c & ((1 << digits) - 1)
  x = np.where(e > 0, (1 + f / 2.0 ** digits) * 2.0 ** (e - bias), f / 2.0 ** digits * 2.0 ** (1 - bias))
  x = np.where(c & 128, -x, x) * 2.0 ** (np.asarray(scale_byte, np.int64) - 127.0)[:, None]
  x[np.asarray(scale_byte) == 255] = np.nan
  return x.reshape(-1)[:len(code)]


def moments32(g, m, v, b1, b2):
  """m', v' of the 8-bit step: separately rounded float32 products and sums."""
  f = np.float32
  g, m, v = (np.asarray(x, f) for x in (g, m, v))
  return m * f(b1) + g * f(1 - b1), v * f(b2) + (g * g) * f(1 - b2)


def encode(x, digits, noise):
  """Codes and scale bytes of float32 values: floor(|x| / spacing + noise), spacing that of the value's binade (or of the
  subnormals) after the block's power of two, in exact float64 arithmetic.  noise: [n] in [0, 1)."""
  n = len(x)
  top, bias = (7, 7) if digits == 3 else (14, 15)
  y, r = _blocks(np.asarray(x, np.float64), n), _blocks(noise, n)
  most = np.abs(y).max(axis=1)
  power = np.where(most > 0, np.frexp(np.where(most > 0, most, 1))[1] - 1 - top, -126).clip(min=-126)
  y = y * 2.0 ** -power[:, None].astype(np.float64)
  e = (np.frexp(y)[1] - 1).clip(min=1 - bias)
  e = np.where(y == 0, 1 - bias, e)
  q = np.floor(np.abs(y) * 2.0 ** (digits - e).astype(np.float64) + r).astype(np.int64)
  code = ((e + bias - 1) << digits) + q          # a carry into the next binade is the next code
  if digits == 2:
    code = np.where((y > 0) & (code == 0), 1, code)
  code = code | (np.signbit(y).astype(np.int64) << 7)
  return code.reshape(-1)[:n].astype(np.uint8), (power + 127).astype(np.uint8)
