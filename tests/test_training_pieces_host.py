"""How the table gradient cuts a token's positions into pieces, compiled for
the host: no position is left out or taken twice up to the largest call."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MOST = 2 ** 31 - 1


@pytest.fixture(scope="module")
def pieces(tmp_path_factory):
    d = tmp_path_factory.mktemp("pieces")
    src, so = d / "p.cpp", d / "p.so"
    src.write_text('#include "pieces.h"\n'
                   'extern "C" int rows_of(int t, int r) { return boa::rows_of_piece(t, r); }\n'
                   'extern "C" int pieces_of(int t, int r) { return boa::pieces_of(t, r); }\n')
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-fsanitize=signed-integer-overflow",
                    "-fsanitize-undefined-trap-on-error", "-I", os.path.join(ROOT, "boa-constrictor_b200", "csrc"),
                    "-o", str(so), str(src)], check=True)
    return C.CDLL(str(so))


@pytest.mark.parametrize("total", [0, 1, 127, 128, 129, 255 * 128, 256 * 128, 256 * 128 + 1, 1 << 20, MOST - 907000,
                                   MOST - 256, MOST - 255, MOST - 1, MOST])
@pytest.mark.parametrize("rows", [128, 160, 906912])
def test_pieces_cover_the_positions_once(pieces, total, rows):
    size, n = pieces.rows_of(total, rows), pieces.pieces_of(total, rows)
    assert size >= rows and 1 <= n <= 256
    assert n == max(1, -(-total // size))
    assert sum(max(0, min(size, total - j * size)) for j in range(n)) == total
    assert n <= total // rows + 1  # what the workspace is laid out for
