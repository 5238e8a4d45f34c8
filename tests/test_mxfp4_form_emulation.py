"""CPU check of the choice between the forms of the product of two MXFP4 operands: tests/emul/emul_gemm4_form.cpp includes the
library's own rule."""
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def form(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    exe = str(tmp_path_factory.mktemp("emul") / "gemm4_form")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-o", exe, os.path.join(ROOT, "tests", "emul", "emul_gemm4_form.cpp")])

    def ask(sizes):
        text = "".join("%d %d %d %d\n" % s for s in sizes)
        out = subprocess.run([exe], input=text, capture_output=True, text=True)
        assert out.returncode == 0, out.stderr
        lines = [tuple(int(v) for v in line.split()) for line in out.stdout.splitlines()]
        assert len(lines) == len(sizes)
        return lines
    return ask


def test_every_form_is_one_the_kernels_take(form):
    """From one SM to 200, from one row to many: tiles that cover the rows, boxes that the copies take, no share of K without work."""
    rng = random.Random(1)
    log = lambda hi: int(2 ** rng.uniform(0, hi))                     # noqa: E731
    sizes = [(M, N, K, sms) for sms in (1, 2, 3, 4, 16, 36, 37, 74, 132, 148, 200) for M in (1, 16, 128, 129, 4096)
             for N, K in ((1, 32), (2048, 2048), (14336, 8192))]
    sizes += [(log(17), log(16), 32 * log(10), rng.randint(1, 200)) for _ in range(3000)]
    for (M, N, K, sms), (ks, tn, mt, tiles) in zip(sizes, form(sizes)):
        assert ks in (0, 1, 2, 4) and tn % 16 == 0 and 16 <= tn <= (128 if ks else 256)
        assert mt * tn >= M > (mt - 1) * tn and tiles == mt * -(-N // (128 if ks else 256))
        assert ks == 0 or mt < 65536
        assert ks < 2 or -(-K // 256) >= 4 * ks


# us on one B200, weights from HBM: one CTA per tile, K split by 2 and 4, CTA pairs with 1 .. 4 more tiles along M than the least
MEASURED = {(16, 4096, 4096): {1: 7.94, 2: 6.44, 4: 6.24, 0: 11.21}, (16, 14336, 4096): {1: 10.0, 2: 13.0, 4: 20.2, 0: 13.3},
            (16, 14336, 8192): {1: 16.0, 2: 20.73, 4: 27.14, 0: 20.83}, (64, 11008, 8192): {1: 14.48, 2: 20.78, 4: 23.06, 0: 18.71},
            (128, 2048, 8192): {1: 12.69, 2: 10.95, 4: 8.92, 0: 15.7}, (16, 28672, 8192): {1: 30.04, 2: 39.09, 4: 48.0, 0: 34.1},
            (256, 4096, 4096): {1: 8.97, 2: 9.1, 4: 15.27, 0: 12.16}, (256, 4096, 14336): {1: 19.02, 2: 15.53, 4: 23.21, 0: 25.19},
            (384, 14336, 2048): {1: 16.59, 2: 33.63, 4: 66.64, 0: 13.85}, (512, 14336, 8192): {1: 47.63, 2: 72.37, 4: 110.89, 0: 34.76},
            (1024, 4096, 4096): {1: 15.98, 2: 30.65, 4: 53.29, 0: 14.21}}
# the pairs' rows per tile, where they are the fastest form: measured with 256, 192, 128 rows per tile 34.8, 41.9, 48.3 us and so on
PAIR_ROWS = {(384, 14336, 2048): 192, (512, 14336, 8192): 256, (1024, 4096, 4096): 256}


def test_form_taken_is_the_fastest_measured(form):
    for size, (ks, tn, _, _) in zip(MEASURED, form([s + (148,) for s in MEASURED])):
        assert MEASURED[size][ks] <= 1.06 * min(MEASURED[size].values()), (size, ks)
        assert ks or tn == PAIR_ROWS[size], (size, tn)


# sizes of tests/test_gpu_mxfp4_forms.py: the form and the rows per tile they are there for
FORMS = {(262, 11008, 32): (0, 96), (289, 11008, 64): (0, 112), (343, 11008, 96): (0, 128), (136, 11008, 288): (0, 144),
         (150, 11008, 544): (0, 160), (180, 11008, 64): (0, 192), (240, 11008, 1056): (0, 240), (500, 11008, 288): (0, 176),
         (512, 14336, 288): (0, 256),
         (1, 20000, 4128): (1, 16), (60, 11008, 4128): (1, 64), (128, 14400, 2080): (1, 128), (33, 2000, 2080): (2, 48),
         (300, 130, 5152): (4, 112), (70, 300, 4128): (4, 80), (16, 4000, 8224): (4, 16)}


def test_sizes_of_the_gpu_test(form):
    got = form([s + (148,) for s in FORMS])
    assert [g[:2] for g in got] == list(FORMS.values())
