"""Host-side checks of the head's operators: the generator's published values, and what is refused without a GPU."""
import ctypes

import numpy as np
import pytest
import torch

import head_oracle as oracle
import l_inf_dist_net_v2_b200 as ldn
from l_inf_dist_net_v2_b200._lib import lib

BAD = 1


def test_the_generator_of_the_oracle_gives_the_published_words():
    for counter, key, want in [
            ([0] * 4, [0] * 2, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
            ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
            ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0], [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1])]:
        assert [int(v) for v in oracle.philox(counter, key)] == want


def test_words_do_not_depend_on_where_they_are_asked_for():
    whole = oracle.words(40, 5, 7)
    assert np.array_equal(whole[6:19], oracle.words(13, 5, 7, first=6))


def test_tensors_on_the_host_are_refused():
    x, w = torch.rand(4, 8), torch.rand(8)
    pair = torch.zeros(3, 8, dtype=torch.int8), torch.ones(3)
    for call in (lambda: ldn.layer_norm(x, w, w), lambda: ldn.dropout(x, 0.1, 1), lambda: ldn.quantize_rows(x),
                 lambda: ldn.dropout_add_layer_norm(x, x, w, w, 0.1, 1), lambda: ldn.layer_norm_quantized(x, w, w),
                 lambda: ldn.int8_linear(x, pair), lambda: ldn.int8_linear((pair[0], pair[1]), pair)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_values_that_make_no_sense_are_refused():
    x = torch.rand(4, 8)
    with pytest.raises(ValueError, match="activation"):
        ldn.int8_linear(x, (x, x), activation="gelu")
    with pytest.raises(ValueError, match="64-bit"):
        ldn.dropout(x, 0.1, -1)
    with pytest.raises(ValueError, match="64-bit"):
        ldn.dropout(x, 0.1, 1, 1 << 64)
    with pytest.raises(ValueError, match="probability"):
        ldn.Dropout(1.5)


def test_the_dropout_layer_keeps_its_place():
    a, b = ldn.Dropout(0.3, seed=5), ldn.Dropout(0.3)
    assert [a.draw() for _ in range(3)] == [(5, 0), (5, 1), (5, 2)]
    b.load_state_dict(a.state_dict())
    assert b.draw() == (5, 3)
    x = torch.rand(2, 3)
    assert b.eval()(x) is x and torch.equal(b(x, x), x + x)


# (whatever stands where a pointer is wanted: none of these calls may launch anything)
@pytest.mark.parametrize("change", [dict(C=0), dict(rows=-1), dict(type=3), dict(eps=float("nan")), dict(eps=-1.0), dict(param_type=1),
                                    dict(x=None), dict(y=None), dict(mean=None)])
def test_layer_norm_arguments(change):
    here = ctypes.create_string_buffer(64)
    a = dict(x=here, pitch=4, rows=2, C=4, type=0, weight=here, bias=here, param_type=0, eps=1e-5, y=here, mean=here, rstd=here, stream=None)
    assert lib.ldn_layer_norm(*{**a, **change}.values()) == BAD


@pytest.mark.parametrize("change", [dict(p=1.5), dict(p=-0.1), dict(p=float("nan")), dict(C=0), dict(type=-1), dict(out=None), dict(rows=-2)])
def test_dropout_arguments(change):
    here = ctypes.create_string_buffer(64)
    a = dict(x=here, pitch=4, residual=None, pitch_residual=0, rows=2, C=4, type=0, p=0.5, seed=1, offset=0, state=None, out=here, stream=None)
    assert lib.ldn_dropout(*{**a, **change}.values()) == BAD


@pytest.mark.parametrize("change", [dict(K=0), dict(K=131072, pitch_q=131072, pitch_w=131072), dict(N=0), dict(M=-1), dict(activation=3),
                                    dict(activation=-1), dict(type=9), dict(pitch_q=3), dict(pitch_w=3), dict(q=None), dict(scale=None),
                                    dict(w=None), dict(w_scale=None), dict(out=None)])
def test_product_arguments(change):
    here = ctypes.create_string_buffer(64)
    a = dict(q=here, pitch_q=16, scale=here, w=here, pitch_w=16, w_scale=here, bias=None, M=2, N=2, K=4, activation=0, out=here, type=0,
             stream=None)
    assert lib.ldn_int8_linear(*{**a, **change}.values()) == BAD


def test_calls_without_rows_do_nothing():
    assert lib.ldn_layer_norm(None, 4, 0, 4, 0, None, None, 0, 1e-5, None, None, None, None) == 0
    assert lib.ldn_dropout(None, 4, None, 0, 0, 4, 0, 0.5, 1, 0, None, None, None) == 0
    assert lib.ldn_quantize_rows(None, 4, 0, 4, 0, None, 16, None, None) == 0
    assert lib.ldn_int8_linear(None, 16, None, None, 16, None, None, 0, 2, 4, 0, None, 0, None) == 0
