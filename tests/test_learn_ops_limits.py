"""Borders of what the learning operators take (bundlesdf_amd/learn_ops.py, the last section of include/nof_hip.h), on the host: what lies behind them is
refused before anything is launched.  Never on a GPU: the addresses are none (tests/conftest.py)."""
import ctypes as C
import os
import subprocess
import sys

import pytest

from bundlesdf_amd import lib

PTR = C.c_void_p(256)                                            # never dereferenced


def refuses(rc):
    return rc < 0 and b'argument check' in lib.load().nof_last_error()


def orthogonalize(*triples):
    """200 x 6 without a workspace: refused in any case, for the coefficients or for that"""
    coef = (C.c_float * (3 * len(triples)))(*[x for t in triples for x in t])
    return lib.load().nof_orthogonalize(PTR, PTR, 0, len(triples), coef, 1e-30, None, 0, 2, 200, 6, None)


def leaves(*triples):
    """in 64 bits, on a grid that is fine enough for the cases below"""
    import numpy as np
    s = np.linspace(0.0, 1.0, 1 << 18)
    with np.errstate(invalid='ignore'):
        for a, b, c in np.float32(triples).astype(float):
            p = a + s * s * (b + s * s * c)
            s = s * p
            if not (np.abs(p).max() <= 15.0 and np.abs(s).max() <= 2.0):
                return True
    return False


def test_coefficients_are_judged_between_any_grid_of_values():
    # 3 / t (s - s^3 / (3 t^2)) has its largest value, 2, at t: here a little more, and less than 2 at every multiple of 1/128
    t = 0.5 + 1 / 256
    peak = (3.0 / t * 1.00002, -1.0 / t ** 3 * 1.00002, 0.0)
    grid = [k / 128 * (peak[0] + (k / 128) ** 2 * peak[1]) for k in range(129)]
    assert max(grid) < 2.0 and leaves(peak)
    so = lib.load()
    assert refuses(orthogonalize(peak)) and b'[0, 2]' in so.nof_last_error()
    lower = (peak[0] * 0.9999, peak[1] * 0.9999, 0.0)
    assert not leaves(lower) and refuses(orthogonalize(lower)) and b'workspace' in so.nof_last_error()      # taken: what is refused is the workspace


@pytest.mark.parametrize('triples', [((3.4445, -4.7750, 2.0315),) * 32, ((1.5, -0.5, 0.0),) * 4, ((3.0, -3.2, 1.2), (2.0, -1.5, 0.5), (1.5, -0.5, 0.0)),
                                     ((0.0, 0.0, 0.0), (15.0, 0.0, 0.0)), ((1.0, 0.0, 0.0),), ((-1.0, 0.0, 0.0), (1.5, -0.5, 0.0)), ((5.0, -20.0, 16.0),) * 6,
                                     ((0.0, 2.0, 0.0),), ((0.0, 0.0, 2.0), (0.5, 0.0, 0.0)), ((8.2872, -23.5959, 17.3004), (4.1071, -2.9478, 0.5448)),
                                     ((2.1, 0.0, 0.0),), ((15.5, -15.0, 0.0),), ((0.0, -2.5, 0.0),), ((1.9, 0.0, 0.0), (0.0, 0.0, 1.0)), ((14.0, -40.0, 27.0),),
                                     ((-1.5, 0.0, 0.0), (1.6, 0.0, 0.0)), ((float('inf'), 0.0, 0.0),), ((1.0, float('nan'), 0.0),), ((1.0, 0.0, float('-inf')),)])
def test_coefficients(triples):
    so = lib.load()
    assert refuses(orthogonalize(*triples))
    assert (b'[0, 2]' in so.nof_last_error()) == leaves(*triples), so.nof_last_error()


def test_embed_gradient_of_more_runs_than_a_launch_holds():
    so = lib.load()

    def bwd(type, N, D):
        return so.nof_embed_bwd(PTR, D, type, PTR, 0, 1.0, PTR, PTR, 1 << 50, N, 4, D, None)

    # bytes of a row: workgroups of the sums, 64 positions a run, 256 threads; a launch holds less than 2^24 of them, 2^22 are the zero role's
    for D, N in ((257, 3 << 29), (512, 3 << 29), (513, 3 << 28), (1 << 20, 3 << 28)):
        assert refuses(bwd(0, N, D)) and b'launches' in so.nof_last_error(), (D, N)
        assert refuses(bwd(1, N, 2 * D)) if 2 * D <= 1 << 20 else True
        assert so.nof_embed_bwd_workspace_bytes(N, 4, 2 * D if 2 * D <= 1 << 20 else D) == -1
        assert so.nof_embed_bwd_workspace_bytes(N - 64, 4, D) > 16 * N
    assert so.nof_embed_bwd_workspace_bytes((1 << 31) - 65537, 4, 256) > 16 << 31


def test_scans_of_more_threads_than_a_launch_holds():
    so = lib.load()
    null = C.c_void_p(None)

    def fwd(t, B, T, D, G):
        return so.nof_gated_scan_fwd(PTR, T * G, G, t, PTR, T * D, D, t, null, null, 0, PTR, PTR, null, PTR, 1 << 50, B, T, D, G, None)

    def bwd(t, B, T, D, G):
        return so.nof_gated_scan_bwd(PTR, T * G, G, t, PTR, T * D, D, t, PTR, T * D, D, null, PTR, null, 0, PTR, PTR, PTR, PTR, 1 << 50, B, T, D, G, None)

    # (type, B, T, D, G): tiles of 64 channels (of two in 16 bits) by one wave; by four; in the backward, a group of two channels is a tile
    for t, B, T, D, G in ((0, 1 << 23, 1, 512, 512), (1, 1 << 23, 1, 1024, 1024), (0, 1 << 21, 64, 512, 1), (0, 1 << 22, 1, 1024, 1024), (2, 1 << 21, 64, 1024, 2)):
        size = so.nof_gated_scan_workspace_bytes
        assert refuses(fwd(t, B, T, D, G)) and refuses(bwd(t, B, T, D, G)), (t, B, T, D, G)
        assert size(B, T, D, G, t) == -1 and so.nof_gated_scan_marks_bytes(B, T, D, G, t) == -1
        assert size(B - 1, T, D, G, t) >= 0
    assert refuses(bwd(1, 1 << 17, 1, 1024, 512)) and so.nof_gated_scan_workspace_bytes(1 << 17, 1, 1024, 512, 1) == 0      # (the forward's)
    assert so.nof_gated_scan_workspace_bytes((1 << 24) - 1, 100000, 1, 1, 0) >= 0                # 256 threads for every B x D: the most


def test_step_of_more_threads_than_a_launch_holds():
    so = lib.load()
    for t, B, D in ((0, 1 << 22, 1024), (0, 1 << 23, 257), (1, 1 << 22, 2048), (2, 1 << 23, 514), (1, 1 << 23, 511), (0, (1 << 24) - 1, 1 << 20)):
        rc = so.nof_gated_scan_step(PTR, D, t, PTR, D, t, PTR, PTR, PTR, B, D, D, None)
        assert refuses(rc) and b'24' in so.nof_last_error(), (t, B, D)


# A library in front of the runtime's: every launch succeeds but the one whose number the environment gives, and the last error is the last call's.
FAKE = r"""
#include <cstdlib>
static int launches, last;
extern "C" int hipLaunchKernel(const void*, ...) { const char* f = getenv("FAIL"); return last = launches++ == (f ? atoi(f) : -1) ? 9 : 0; }
extern "C" int hipGetLastError() { const int e = last; last = 0; return e; }
extern "C" int __hipPushCallConfiguration(...) { return 0; }
extern "C" int __hipPopCallConfiguration(...) { return 0; }
extern "C" int hipFuncSetAttribute(const void*, int, int) { return 0; }
extern "C" int fake_launches() { return launches; }
"""
CALLS = """
import ctypes as C, sys
fake = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
so = C.CDLL(sys.argv[2])
p, null, i64, f = C.c_void_p(256), C.c_void_p(None), C.c_int64, C.c_float
quintic = (f * 15)(*[3.4445, -4.7750, 2.0315] * 5)
ws = i64(1 << 40)
call = {
    'gradient': lambda: so.nof_embed_bwd(p, i64(8), 0, p, 0, f(1.0), p, p, ws, i64(9000), i64(70000), 8, null),
    'small gradient': lambda: so.nof_embed_bwd(p, i64(8), 0, p, 0, f(1.0), p, p, ws, i64(900), i64(70000), 8, null),
    'scan': lambda: so.nof_gated_scan_fwd(p, i64(9000), i64(1), 0, p, i64(9000 * 4), i64(4), 0, null, null, 0, p, p, null, p, ws, i64(1), i64(9000), 4, 1, null),
    'scan back': lambda: so.nof_gated_scan_bwd(p, i64(9000), i64(1), 0, p, i64(9000 * 200), i64(200), 0, p, i64(9000 * 200), i64(200), null, p, null, 0, p, p, p,
                                               p, ws, i64(1), i64(9000), 200, 1, null),
    'update': lambda: so.nof_orthogonalize(p, p, 0, 5, quintic, f(1e-30), p, ws, i64(1), i64(200), i64(300), null),
    'cut update': lambda: so.nof_orthogonalize(p, p, 1, 5, quintic, f(1e-30), p, ws, i64(1), i64(200), i64(2000), null),
    'thin update': lambda: so.nof_orthogonalize(p, p, 2, 5, quintic, f(1e-30), p, ws, i64(1), i64(90), i64(2000), null),
}[sys.argv[3]]
print(call(), fake.fake_launches())
"""


@pytest.mark.parametrize('call,launches', [('gradient', 6), ('small gradient', 3), ('scan', 2), ('scan back', 3), ('update', 17), ('cut update', 22), ('thin update', 7)])
def test_a_launch_that_fails_is_the_last_and_reported(tmp_path, call, launches):
    fake = tmp_path / 'libfake.so'
    (tmp_path / 'fake.cpp').write_text(FAKE)
    subprocess.run(['g++', '-shared', '-fPIC', '-o', str(fake), str(tmp_path / 'fake.cpp')], check=True)
    lib.load()

    def run(fail):
        r = subprocess.run([sys.executable, '-c', CALLS, str(fake), lib.LIB_PATH, call], env={**os.environ, 'FAIL': str(fail)}, capture_output=True, text=True, check=True)
        return tuple(int(x) for x in r.stdout.split())

    assert run(-1) == (0, launches)
    for k in range(launches):
        assert run(k) == (9, k + 1), k
