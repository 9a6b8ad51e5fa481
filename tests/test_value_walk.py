"""Waits of the dv kernel's loading and issuing lane, replayed on the host from the kernel's own source
(tests/host/value_walk.cpp): every product waits for what it reads and overwrites, whatever tiles a CTA gets one after
the other, and however early or late the barriers complete."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CXX = os.environ.get('CXX') or shutil.which('g++')

pytestmark = pytest.mark.skipif(not CXX, reason='no C++ compiler')

# CTAs, B, H, T, S, w, lengths (repeated over the batch)
PROBLEMS = [
    ('148', 200, 1, 128, 384, 64),                      # tiles nobody sees between tiles of one step
    ('148', 64, 8, 64, 1000, 128, 700, 333, 128, 1000, 90),
    ('148', 64, 1, 1, 1024, 256),
    ('148', 64, 12, 100, 100, 64, 100, 0, 0, 57),       # batches without keys
    ('148', 200, 1, 256, 256, 1, 256, 100, 0),
    ('148', 8, 40, 128, 128, 64, 128, 128, 0),
    ('148', 16, 16, 100, 300, 256, 300, 150, 110, 300),
    ('148', 16, 16, 64, 1500, 256),
    ('148', 8, 4, 2047, 2047, 128, 2047, 1500, 700, 1001),
    ('148', 2, 16, 4096, 4096, 256),
]


@pytest.fixture(scope='module')
def replay(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp('walk') / 'value_walk')
    res = subprocess.run([CXX, '-O2', '-std=c++17', '-I', os.path.join(ROOT, 'fly_b200', 'csrc'),
                          os.path.join(ROOT, 'tests', 'host', 'value_walk.cpp'), '-o', exe],
                         stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert res.returncode == 0, res.stdout

    def run(*args):
        res = subprocess.run([exe, *map(str, args)], stdout=subprocess.PIPE, text=True, timeout=300)
        assert res.returncode == 0, res.stdout

    return run


@pytest.mark.parametrize('problem', PROBLEMS, ids=lambda p: '-'.join(map(str, p[1:6])))
def test_every_product_waits(replay, problem):
    replay(*problem)


def test_small_problems_in_every_order(replay):
    replay('random', 3000)
