"""The tensor-core kernels of attention and its gradients, run on the host from their own source under random schedules
(tests/host/model): warps, loads, products and stores at speeds that differ by up to a thousand.  The results are those of
the definition in 64 bits, and the same bits under every schedule: a wait that is missing, or that can pass too early,
shows as a difference, as what was never written, or as a schedule in which nothing can go on.

Tolerance: that of test_training_gpu.py, 3 * 2^-8 in the 2-norm (the models' products are exact sums in fp32, as the tensor
core's are up to their order)."""
import concurrent.futures
import os
import re
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MODEL = os.path.join(ROOT, 'tests', 'host', 'model')
sys.path.insert(0, MODEL)
CXX = os.environ.get('CXX') or shutil.which('g++')
CUDA = os.environ.get('CUDA_HOME', '/usr/local/cuda')
TOL = 3 * 2.0 ** -8

pytestmark = pytest.mark.skipif(
    not CXX or not os.path.exists(os.path.join(CUDA, 'include', 'cuda_bf16.h')) or os.uname().machine != 'x86_64',
    reason='needs a C++ compiler, the CUDA headers and x86-64')


def build(out, change=lambda name, text: text):
    from translate import write_units
    out = str(out)
    units = write_units(os.path.join(ROOT, 'fly_b200', 'csrc'), out, change)
    sources = units + [os.path.join(MODEL, n) for n in ('device_model.cpp', 'driver.cpp')]
    jobs = []
    for src in sources:
        obj = os.path.join(out, os.path.basename(src) + '.o')
        cmd = [CXX, '-O2', '-std=c++17', '-w', '-ffp-contract=off', '-I', MODEL, '-I', os.path.join(ROOT, 'include'),
               '-I', os.path.join(CUDA, 'include'), '-c', src, '-o', obj]
        if src.endswith('device_model.cpp'):
            cmd.insert(1, '-O3')
        jobs.append((obj, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    for obj, job in jobs:
        log = job.communicate()[0]
        assert job.returncode == 0, log
    exe = os.path.join(out, 'driver')
    # (the kernels for any shape are not linked: nothing here calls them)
    res = subprocess.run([CXX, '-no-pie', '-o', exe, *(obj for obj, _ in jobs), '-Wl,--unresolved-symbols=ignore-all'],
                         stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert res.returncode == 0, res.stdout
    return exe


@pytest.fixture(scope='module')
def driver(tmp_path_factory):
    return build(tmp_path_factory.mktemp('model'))


def run(exe, problem, schedules, first=0):
    B, H, T, S, D, w, sms, *lengths = problem
    args = [5, B, H, T, S, D, w, sms, schedules, first, *lengths]
    return subprocess.run([exe, *map(str, args)], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=600)


def check(res):
    assert res.returncode == 0, res.stdout
    errors = [float(x) for x in re.findall(r'(?:out|dq|dk|dv) (\S+)', res.stdout)]
    assert len(errors) == 4 and all(e <= TOL for e in errors), res.stdout
    assert ', 0 differ' in res.stdout, res.stdout


# B, H, T, S, head dim, w, SMs, lengths
PROBLEMS = [
    (1, 1, 300, 300, 64, 64, 1),
    (2, 1, 300, 300, 128, 100, 1),
    (4, 2, 180, 27, 64, 214, 1),                     # query tiles of one key tile each
    (8, 1, 64, 384, 64, 64, 2),                      # key tiles of one step, and some that nobody sees
    (4, 1, 64, 384, 128, 64, 1),
    (6, 1, 100, 100, 64, 64, 1, 100, 0, 0, 57),      # batches without keys
    (4, 1, 100, 100, 128, 64, 1, 100, 0, 57, 0),
    (2, 2, 257, 257, 64, 1, 2),
    (1, 2, 129, 500, 64, 700, 1, 444),
    (1, 1, 500, 129, 128, 300, 1),
    (3, 1, 1, 300, 64, 16, 1),
]


def test_results_do_not_depend_on_the_schedule(driver):
    with concurrent.futures.ThreadPoolExecutor(os.cpu_count()) as pool:
        for res in pool.map(lambda p: run(driver, p, 5), PROBLEMS):
            check(res)


# a wait less in a copy of the source, and a problem that needs it
MISTAKES = [
    ('sbl_bwd_walk.cuh', 'v.minus(t, it, s, n, pend_s >= 0);', 'v.minus(t, it, s, n, n > 0);', (8, 1, 64, 384, 64, 64, 2)),
    ('sbl_band_walk.cuh', 'if (last >= 0 && last >= g - 2) mbar_wait(', 'if (false) mbar_wait(', (4, 2, 180, 27, 64, 214, 1)),
]


@pytest.mark.parametrize('mistake', MISTAKES, ids=lambda m: m[0])
def test_a_missing_wait_is_seen(mistake, tmp_path):
    """The models can tell: without one of its waits the same source fails here."""
    name, good, bad, problem = mistake

    def change(file, text):
        if file != name:
            return text
        assert text.count(good) == 1
        return text.replace(good, bad)

    exe = build(tmp_path, change)
    with concurrent.futures.ThreadPoolExecutor(os.cpu_count()) as pool:
        results = list(pool.map(lambda first: run(exe, problem, 5, first), range(0, 60, 5)))
    assert any(r.returncode == 3 or ', 0 differ' not in r.stdout or 'nan' in r.stdout for r in results)
