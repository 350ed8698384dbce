"""Whether rows of two tensors share memory (csrc/rows.h), and the calls that are refused for it, with no GPU."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # (an aligned address, refused before it is used)

SHIM = """
#include "rows.h"
extern "C" int meet(const long* a, const long* b) {
  const nkl::Rows x{(size_t)a[0], a[1], a[2], a[3], a[4], a[5]}, y{(size_t)b[0], b[1], b[2], b[3], b[4], b[5]};
  return nkl::rows_meet(x, y);
}
extern "C" int share(const long* a) {
  return nkl::rows_share(nkl::Rows{(size_t)a[0], a[1], a[2], a[3], a[4], a[5]});
}
"""


@pytest.fixture(scope="module")
def rows(tmp_path_factory):
    cc = shutil.which("g++")
    if cc is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("rows")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run([cc, "-O1", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "nki-kernel-lab_amd", "csrc"),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True, timeout=120)
    lib = ctypes.CDLL(str(d / "shim.so"))
    pack = lambda t: (ctypes.c_long * 6)(*t)  # noqa: E731
    return lambda a, b: bool(lib.meet(pack(a), pack(b))), lambda a: bool(lib.share(pack(a)))


def held(t):
    at, H, S, sh, ss, n = t
    return [at + h * sh + s * ss + i for h in range(H) for s in range(S) for i in range(n)]


def test_against_sets(rows):
    """Exact where rows are as far apart in both, never too lax elsewhere."""
    meet, share = rows
    rng = random.Random(0)
    exact = 0
    for _ in range(20000):
        ss = rng.randrange(0, 40)
        tensors = [(1000 + rng.randrange(0, 60), rng.randrange(1, 5), rng.randrange(1, 5), rng.randrange(0, 60),
                    ss if rng.random() < 0.8 else rng.randrange(0, 40), rng.randrange(1, 9)) for _ in range(2)]
        a, b = tensors
        sets = [held(t) for t in tensors]
        common = bool(set(sets[0]) & set(sets[1]))
        if a[2] == 1 or b[2] == 1 or a[4] == b[4]:
            assert meet(a, b) == common, (a, b)
            exact += common
        else:
            assert meet(a, b) or not common, (a, b)
        assert meet(a, b) == meet(b, a)
        assert share(a) == (len(set(sets[0])) < len(sets[0])), a
    assert 1000 < exact < 19000
    assert not meet((1000, 0, 3, 8, 8, 8), (1000, 1, 1, 0, 0, 8)) and not share((1000, 3, 0, 0, 0, 8))


def test_columns_of_a_projection(rows):
    meet, share = rows
    S, row = 50, 12 * 128
    q, k = (0, 8, S, 128, row, 128), (8 * 128, 2, S, 128, row, 128)
    assert not meet(q, k) and not meet(k, q) and not share(q)
    assert meet(q, (7 * 128 + 1, 2, S, 128, row, 128)) and meet(q, (2, 8, S, 128, row, 128))


def test_products_refuse_outputs_over_their_operands():
    from nkilab import _lib

    def call(x=P, y=P + (1 << 16), r=None, M=4, N=128, K=128, ldx=128, ldy=128, ldr=128, dt=1, do=1):
        rc = _lib.lib().nkl_gemm_w4(x, P + (1 << 18), P + (1 << 19), None, y, r, M, N, K, 64, ldx, ldy, ldr, 0, dt, dt, do, None)
        return rc == -1 and b"share memory" in _lib.lib().nkl_last_error_string()

    for bad in (dict(y=P), dict(y=P + 2), dict(y=P + 1022), dict(y=P - 1022), dict(ldx=256, ldy=256, y=P + 254),
                dict(M=1, y=P), dict(do=0, y=P + 1020), dict(ldx=200, y=P + 300),
                dict(r=P + (1 << 16) + 2), dict(r=P + (1 << 16), ldr=256), dict(r=P + (1 << 16) - 256, M=2)):
        assert call(**bad), bad


def test_rotations_refuse_outputs_over_their_inputs():
    from nkilab import _lib, ops

    L, r = _lib.lib(), ops.Rotary(64)._packed

    def rotate(y, st=(64, 128, 64, 128), H=2, S=3):
        rc = L.nkl_rotary_apply(r, P, y, H, S, 64, *st, None, 0, 0, 0, 0, None)
        return rc == -1 and b"share memory" in L.nkl_last_error_string()

    for bad in (dict(y=P + 4), dict(y=P - 4), dict(y=P + 256), dict(y=P + 2 * 512), dict(y=P + 16, H=1, S=1),
                dict(y=P + 128, st=(192, 64, 64, 128)), dict(y=P + 65536, st=(64, 128, 64, 64)),
                dict(y=P + 65536, st=(64, 128, 32, 128)), dict(y=P + 65536, st=(64, 128, 96, 32))):
        assert rotate(**bad), bad


def test_appends_refuse_q_out_over_what_they_read():
    from test_cache8_host import d8, scales

    from nkilab import _lib, ops

    L, r = _lib.lib(), ops.Rotary(64)._packed

    def write(q=P, qo=P + 65536, k=P + (1 << 18), v=P + (1 << 19), so=(256, 64)):
        rc = L.nkl_cache_write(ctypes.byref(d8()), scales(v=P + 4096), k, v, 256, 64, 256, 64, q, qo, 4, 256, 64, *so, None, 0, r,
                               1, None)
        return rc == -1 and b"share memory" in L.nkl_last_error_string()

    for bad in (dict(qo=P + 64), dict(qo=P + 2), dict(k=P + 65536), dict(v=P + 65536 + 128), dict(so=(200, 64)), dict(so=(256, 32))):
        assert write(**bad), bad
