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
