"""The 16-bit code that a slope of an activation is kept in (`Slope16` in mineral_amd/csrc/linear_act.hip), restated with numpy: its fourth
root in steps of 1/30720.  CPU only: this pins the bounds that the kernel's comment states, tests/test_linear_act_gradient.py the kernel."""
import numpy as np

STEPS = np.float32(30720)
BACK = np.float32(1 / 30720.0 ** 4)


def pack(s):
    a = np.abs(s)
    q = np.sqrt(np.sqrt(a))
    u = np.floor(np.where(a < 1.25, q, 0).astype(np.float64) * 30720 + 0.5).astype(np.int64)
    return np.where(a < 1.25, u, 0x7FFF) | np.where(np.signbit(s), 0x8000, 0)


def unpack(u):
    q = (u & 0x7FFF).astype(np.float32)
    a = q * q
    a = a * a * BACK
    return np.where((u & 0x7FFF) == 0x7FFF, np.float32(np.nan), np.where(u & 0x8000, -a, a)).astype(np.float32)


def samples():
    rng = np.random.default_rng(1)
    s = np.exp2(rng.uniform(-62, np.log2(1.2), 2000000)).astype(np.float32)
    return s * np.where(rng.random(s.size) < 0.5, np.float32(-1), np.float32(1))


def test_every_code_is_its_own_slope():
    u = np.arange(0x7FFF)
    u = u[unpack(u) < 1.25]
    assert u[-1] > 32000 and np.array_equal(pack(unpack(u)), u)


def test_error_over_all_magnitudes():
    s = samples()
    err = np.abs(unpack(pack(s)).astype(np.float64) - s)
    q = np.abs(s.astype(np.float64)) ** 0.25
    assert np.all(err <= (q + 0.5 / 30720) ** 4 - q ** 4 + 2.0 ** -20 * np.abs(s))
    rel = err / np.abs(s)
    for low, high, most in ((2.0 ** -2, 1.2, -13.4), (2.0 ** -4, 1.2, -12.9), (2.0 ** -14, 1.2, -10.4), (2.0 ** -16, 1.2, -9.9), (2.0 ** -24, 1.2, -7.9), (2.0 ** -40, 1.2, -3.8)):
        at = (np.abs(s) >= low) & (np.abs(s) < high)
        assert rel[at].max() <= 2.0 ** most, (low, np.log2(rel[at].max()))


def test_zero_one_and_what_is_no_slope():
    assert unpack(pack(np.float32([0.0, -0.0, 1.0, -1.0]))).tolist() == [0.0, 0.0, 1.0, -1.0]
    assert np.all(np.isnan(unpack(pack(np.float32([np.nan, np.inf, -np.inf, 1.25, 3.4e38])))))
    assert np.all(unpack(pack(np.float32([2.0 ** -63, 2.0 ** -60]))) > 0) and unpack(pack(np.float32([2.0 ** -66])))[0] == 0
