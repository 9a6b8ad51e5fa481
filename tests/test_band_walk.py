"""The head-dim-64 band kernel's phi(K) slots, replayed on the host from the kernel's own source (tests/host/band_walk.cpp):
no slot is filled while a product may still read it, whatever query tiles a CTA gets one after the other."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CXX = os.environ.get('CXX') or shutil.which('g++')

pytestmark = pytest.mark.skipif(not CXX, reason='no C++ compiler')

# CTAs, B, H, T, S, w, lengths (repeated over the batch)
PROBLEMS = [
    ('148', 21, 11, 177, 27, 214),                      # two query tiles, one key tile
    ('148', 94, 2, 144, 74, 252, 56, 74, 34, 74, 57, 74),
    ('148', 17, 14, 181, 15, 669, 2, 8, 0, 13),
    ('148', 32, 8, 512, 512, 128, 100, 90, 512, 128),   # short texts in a padded batch
    ('148', 64, 4, 700, 100, 2048),
    ('148', 200, 1, 128, 384, 64),
    ('148', 8, 1, 196, 196, 256),
    ('148', 8, 4, 2047, 2047, 128, 2047, 1500, 700, 1001),
    ('148', 2, 8, 8192, 8192, 256),
]


@pytest.fixture(scope='module')
def replay(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp('walk') / 'band_walk')
    res = subprocess.run([CXX, '-O2', '-std=c++17', '-I', os.path.join(ROOT, 'fly_b200', 'csrc'),
                          '-I', os.path.join(ROOT, 'include'),
                          os.path.join(ROOT, 'tests', 'host', 'band_walk.cpp'), '-o', exe],
                         stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert res.returncode == 0, res.stdout

    def run(*args):
        res = subprocess.run([exe, *map(str, args)], stdout=subprocess.PIPE, text=True, timeout=300)
        assert res.returncode == 0, res.stdout

    return run


@pytest.mark.parametrize('problem', PROBLEMS, ids=lambda p: '-'.join(map(str, p[1:6])))
def test_no_slot_is_filled_too_early(replay, problem):
    replay(*problem)


def test_small_problems(replay):
    replay('random', 4000)
