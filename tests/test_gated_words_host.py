"""The rule by which the gated projection's copies read pieces of 16-bit rows that start anywhere, compiled for the host: every word that it
reads has to lie in the tensor's memory."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def words_of_piece(tmp_path_factory):
    at = tmp_path_factory.mktemp("words")
    source, built = at / "words.cpp", at / "words.so"
    source.write_text('#include "ldn_words.cuh"\n'
                      'extern "C" int words(unsigned off, int c, int C, long long row, long long rows, long long pitch) {\n'
                      '    return ldn::words_of_piece(off, c, C, row, rows, pitch);\n}\n')
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "l_inf_dist_net_v2_b200", "csrc"), str(source), "-o",
                    str(built)], check=True)
    f = ctypes.CDLL(str(built)).words
    f.argtypes = [ctypes.c_uint, ctypes.c_int, ctypes.c_int, ctypes.c_longlong, ctypes.c_longlong, ctypes.c_longlong]
    return f


# (a repeated row, windows that overlap, rows side by side, rows with a gap)
@pytest.mark.parametrize("pitch_of", [lambda C: 0, lambda C: 1, lambda C: 3, lambda C: 7, lambda C: 8, lambda C: 13, lambda C: C - 1, lambda C: C,
                                      lambda C: C + 1, lambda C: C + 5, lambda C: 2 * C + 8])
def test_what_is_read_lies_in_the_tensor(words_of_piece, pitch_of):
    for C in (1, 7, 8, 9, 15, 16, 17, 23, 24, 25, 40, 41, 104):
        pitch = max(0, pitch_of(C))
        for rows in (1, 2, 3, 9):
            for start in range(8):  # elements in front of the tensor in its 16 bytes
                begin, end = 2 * start, 2 * (start + (rows - 1) * pitch + C)
                for row in range(rows):
                    for c in range(0, C, 8):
                        at = 2 * (start + row * pitch + c)
                        off, words = at % 16, words_of_piece(at % 16, c, C, row, rows, pitch)
                        if words == 0:
                            continue
                        # the piece is whole and comes of what is read
                        assert c + 8 <= C and (words == 2 or off == 0)
                        assert begin <= at - off and at - off + 16 * words <= end, (C, pitch, rows, start, row, c)


def test_rows_side_by_side_are_read_as_words(words_of_piece):
    """All but the pieces at the tensor's two ends and the rows' cut ends."""
    rows, C = 5, 41
    alone = [(row, c) for row in range(rows) for c in range(0, C - 7, 8) if not words_of_piece(2 * (row * C + c) % 16, c, C, row, rows, C)]
    assert alone == [(rows - 1, 32)]
