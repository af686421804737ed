"""The partial sums that the cross entropy's gradients add up are those that their launches write, from the
launches' own arguments (tests/native/head_parts.hip)."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FP32, BF16, FP16 = 0, 1, 2


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    at = str(tmp_path_factory.mktemp("head_parts"))
    obj, exe = os.path.join(at, "head_parts.o"), os.path.join(at, "head_parts")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "--offload-host-only", "-O1", "-std=c++17", "-Wno-unused-function",
                    "-I", os.path.join(ROOT, "include"), "-c", os.path.join(ROOT, "tests", "native", "head_parts.hip"),
                    "-o", obj], check=True)
    subprocess.run([HIPCC, obj, "-o", exe], check=True)

    def run(shapes):
        text = "".join("%d %d %d %d\n" % s for s in shapes)
        out = subprocess.run([exe], input=text, capture_output=True, text=True, timeout=300, check=True).stdout
        lines = [line.split(": ") for line in out.splitlines()]
        assert [line[0] for line in lines] == [line.strip() for line in text.splitlines()]
        return [line[1].split() for line in lines]

    return run


def check(shape, words):
    assert words[-2:] == ["outside", "0"], shape
    written = {"dx": 0, "dw": 0}
    summed = {"dx": 0, "dw": 0}
    for word in words[:-2]:
        which, sign, count = word[:2], word[2], int(word[3:])
        if sign == "+" and which == "dw":
            assert not written["dw"] or summed["dw"] or written["dw"] == count, (shape, words)
            written["dw"], summed["dw"] = count, 0
        elif sign == "+":
            # each piece adds to the first ones' sums, and begins none
            assert not written["dx"] or count <= written["dx"], (shape, words)
            written["dx"] = max(written["dx"], count)
        else:
            assert count == written[which], (shape, words)
            summed[which] = count
    assert written == summed, (shape, words)


def test_named_shapes(launches):
    """Sizes whose classes end some ranges before the multiple of 256 that a piece is filled up to."""
    shapes = [(t, *s) for t in (FP32, BF16, FP16) for s in (
        (512, 50000, 128), (512, 50000, 256), (1024, 9250, 128), (1024, 9250, 256), (512, 9250, 512), (743, 14141, 128),
        (4, 41171, 128), (282, 25354, 165), (100, 33537, 128), (100, 33600, 128), (4096, 65536, 1024), (4096, 10007, 128),
        (8300, 4200, 24), (16384, 40000, 64), (9000, 24001, 24), (8200, 40500, 24), (16384, 139310, 16), (1 << 20, 16400, 16), (1, 1, 1), (64, 1000, 128))]
    for shape, words in zip(shapes, launches(shapes)):
        check(shape, words)


def test_many_shapes(launches):
    r = random.Random(1)
    spread = lambda most: min(most, int(2 ** r.uniform(0, most.bit_length())) + r.randrange(9))  # noqa: E731
    shapes = [(r.randrange(3), max(1, spread(1 << 20)), max(1, spread(1 << 20)),
               max(1, r.choice([128, spread(4096), 8 * spread(512)]))) for _ in range(40000)]
    for rows in range(256, 2100, 256):
        for classes in range(5000, 60000, 61):
            shapes.append((rows // 256 % 2, rows, classes, r.choice([128, 256, 512])))
    parts = 0
    for shape, words in zip(shapes, launches(shapes)):
        check(shape, words)
        parts += any(w.startswith("dx=") for w in words)
    assert parts > len(shapes) // 4


def test_pieces(launches):
    """How many pieces tests/test_gpu_cross_entropy_pieces.py takes, so that it keeps testing several."""
    shapes = [(t, *s) for t in (FP32, BF16) for s in ((9000, 24001, 24), (8200, 40500, 24), (16384, 139310, 16))]
    counts = [[int(w[3:]) for w in words if w.startswith("dx+")] for words in launches(shapes)]
    assert [len(c) for c in counts] == [2, 3, 17] * 2
    assert all(c[-1] < c[0] for c in counts[2::3])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("classes,width", [(10, 8), (1 << 18, 1 << 15), ((1 << 18) + 1, 1 << 15), (1 << 20, 1 << 16)])
def test_no_rows_take_no_workspace(mg, dtype, classes, width):
    """Zeros in dW are all that there is to write."""
    assert mg.cross_entropy_backward_workspace(0, classes, width, dtype) == 0
