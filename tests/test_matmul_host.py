"""The 4-bit products, routing and combine refuse bad arguments before touching a GPU."""

import pytest
import torch

from chad_b200 import _lib, experts, ops

OK, EINVAL, EUNSUP, EWS, EALIGN = (_lib.QKV_OK, _lib.QKV_EINVAL, _lib.QKV_EUNSUPPORTED,
                                   _lib.QKV_EWORKSPACE, _lib.QKV_EALIGN)


def _matmul(lib, **over):
    a = dict(x=16, ldx=256, w=16, s=16, b=16, out=1 << 20, M=4, N=32, K=256, bits=4, gs=64, dtype=0,
             act=0, ws=16, ws_bytes=1 << 30, stream=None)
    a.update(over)
    return lib.qkv_quantized_matmul(*a.values())


@pytest.mark.parametrize("over,code", [
    (dict(bits=8), EUNSUP), (dict(bits=3), EUNSUP), (dict(gs=32), EUNSUP), (dict(dtype=2), EINVAL),
    (dict(act=2), EINVAL), (dict(act=-1), EINVAL), (dict(M=-1), EINVAL), (dict(N=0), EINVAL),
    (dict(K=0, ldx=0), EINVAL), (dict(K=96), EINVAL), (dict(N=31, act=1), EINVAL),
    (dict(ldx=248), EINVAL), (dict(ldx=260), EALIGN), (dict(x=8), EALIGN), (dict(w=4), EALIGN),
    (dict(s=17), EALIGN), (dict(out=1), EALIGN), (dict(x=None), EINVAL), (dict(w=None), EINVAL),
    (dict(s=None), EINVAL), (dict(b=None), EINVAL), (dict(out=None), EINVAL), (dict(M=0), OK),
    # x ends at 16 + 4 * 512, out is 4 * 64 bytes long
    (dict(out=16), EINVAL), (dict(out=14 + 4 * 512), EINVAL), (dict(x=1024, out=770), EINVAL),
])
def test_matmul_rejects_bad_arguments(over, code):
    lib = _lib.load()
    assert _matmul(lib, **over) == code
    if code != OK:
        assert lib.qkv_last_error()


def _grouped(lib, **over):
    a = dict(x=16, ldx=256, x_rows=8, rows=None, offsets=16, w=16, s=16, b=16, out=1 << 20, R=8,
             E=4, N=32, K=256, bits=4, gs=64, dtype=0, act=0, ws=16, ws_bytes=1 << 30, stream=None)
    a.update(over)
    return lib.qkv_grouped_matmul(*a.values())


@pytest.mark.parametrize("over,code", [
    (dict(offsets=None), EINVAL), (dict(R=9), EINVAL), (dict(E=0), EINVAL), (dict(bits=2), EUNSUP),
    (dict(offsets=18), EALIGN), (dict(rows=18), EALIGN), (dict(x_rows=-1), EINVAL),
    (dict(K=100, ldx=104), EINVAL), (dict(R=0, x_rows=0), OK), (dict(out=16), EINVAL),
])
def test_grouped_rejects_bad_arguments(over, code):
    assert _grouped(_lib.load(), **over) == code


def _route(lib, **over):
    a = dict(logits=16, dtype=0, T=4, E=64, k=8, normalize=1, experts=16, weights=16, rows=16,
             slots=16, offsets=16, ws=16, ws_bytes=1 << 30, stream=None)
    a.update(over)
    return lib.qkv_route_topk(*a.values())


@pytest.mark.parametrize("over,code", [
    (dict(k=0), EINVAL), (dict(k=65), EINVAL), (dict(k=17), EUNSUP), (dict(E=513), EUNSUP),
    (dict(E=0), EINVAL), (dict(T=-1), EINVAL), (dict(dtype=3), EINVAL), (dict(logits=None), EINVAL),
    (dict(offsets=None), EINVAL), (dict(experts=None), EINVAL), (dict(weights=18), EALIGN),
    (dict(logits=17), EALIGN), (dict(T=1000, ws=None), EWS), (dict(T=1000, ws_bytes=64), EWS),
    (dict(T=1000, ws=20), EALIGN), (dict(T=(1 << 24) + 1), EUNSUP),
])
def test_route_rejects_bad_arguments(over, code):
    assert _route(_lib.load(), **over) == code


def _combine(lib, **over):
    a = dict(y=16, R=32, slots=16, weights=16, residual=None, out=1 << 20, T=4, k=8, N=64, dtype=0,
             stream=None)
    a.update(over)
    return lib.qkv_expert_combine(*a.values())


@pytest.mark.parametrize("over,code", [
    (dict(dtype=2), EINVAL), (dict(T=-1), EINVAL), (dict(k=0), EINVAL), (dict(N=0), EINVAL),
    (dict(y=None), EINVAL), (dict(slots=None), EINVAL), (dict(out=None), EINVAL),
    (dict(out=8), EALIGN), (dict(residual=8), EALIGN), (dict(T=0), OK),
    (dict(out=16), EINVAL), (dict(out=32 * 128), EINVAL),
    (dict(residual=(1 << 20) + 16), EINVAL), (dict(residual=(1 << 20) - 16), EINVAL),
])
def test_combine_rejects_bad_arguments(over, code):
    assert _combine(_lib.load(), **over) == code


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.qkv_route_workspace_size(0, 64) == 0
    assert lib.qkv_route_workspace_size(64, 64) == 0
    # two counts to a word; blocks of 32 tokens, then larger ones so that 256 are not passed
    assert lib.qkv_route_workspace_size(65, 64) == 3 * 32 * 4
    assert lib.qkv_route_workspace_size(8192, 128) == 256 * 64 * 4
    assert lib.qkv_route_workspace_size(8193, 128) == 129 * 64 * 4
    assert lib.qkv_route_workspace_size(65, 7) == 3 * 4 * 4


def test_operators_refuse_cpu_tensors():
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    w = (torch.zeros(16, 16, dtype=torch.int32), torch.zeros(16, 2, dtype=torch.bfloat16),
         torch.zeros(16, 2, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        ops.quantized_matmul(x, w)
    with pytest.raises(ValueError):
        ops.grouped_quantized_matmul(x, tuple(t[None] for t in w), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        ops.route_topk(torch.zeros(2, 8), 2)
    with pytest.raises(ValueError):
        ops.expert_combine(x, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1))


def test_layers_check_their_shapes():
    with pytest.raises(ValueError):
        experts.quantize_weight(torch.zeros(4, 100))
    e = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    up = (e(4, 128, 16, dt=torch.int32), e(4, 128, 2), e(4, 128, 2))      # F 64, K 128
    down = (e(4, 128, 8, dt=torch.int32), e(4, 128, 1), e(4, 128, 1))
    experts.QuantizedExperts(up, down, 2)
    with pytest.raises(ValueError):
        experts.QuantizedExperts(up, up, 2)
    with pytest.raises(ValueError):
        experts.QuantizedExperts(up, down, 5)


def test_python_bindings_return_the_librarys_codes():
    ext = _lib.ext()
    assert ext.quantized_matmul(16, 256, 16, 16, 16, 16, 4, 32, 96, 4, 64, 0, 0, None, 0, None) == EINVAL
    assert ext.grouped_matmul(16, 256, 8, None, None, 16, 16, 16, 16, 8, 4, 32, 256, 4, 64, 0, 0,
                              None, 0, None) == EINVAL
    assert ext.route_topk(16, 0, 4, 64, 0, 1, 16, 16, 16, 16, 16, None, 0, None) == EINVAL
    assert ext.expert_combine(16, 32, 16, 16, None, 16, 4, 8, 64, 2, None) == EINVAL
    with pytest.raises(TypeError):
        ext.route_topk(16)


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch on addresses that are none")
@pytest.mark.parametrize("call", [_matmul, _grouped, _route, _combine])
def test_a_refused_launch_names_the_cuda_error(call):
    lib = _lib.load()
    assert call(lib) == _lib.QKV_ECUDA
    message = lib.qkv_last_error().decode()
    assert "unsupported" not in message and "launch failed" not in message
    assert message.startswith("qkv_"), message


@pytest.mark.parametrize("x,logits", [((3, 128), (2, 4)), ((2, 128), (3, 4)), ((1, 2, 128), (2, 4)),
                                      ((2, 128), (4,))])
def test_experts_layer_refuses_logits_of_other_tokens(x, logits):
    e = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    layer = experts.QuantizedExperts((e(4, 128, 16, dt=torch.int32), e(4, 128, 2), e(4, 128, 2)),
                                     (e(4, 128, 8, dt=torch.int32), e(4, 128, 1), e(4, 128, 1)), 2)
    with pytest.raises(ValueError, match="same tokens"):
        layer(e(*x), e(*logits))


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch on addresses that are none")
@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 16, 2 ** 31 - 256])
def test_products_refuse_rows_whose_tiles_pass_32_bits(n):
    lib = _lib.load()
    far = 1 << 50  # out behind every other range
    assert _matmul(lib, M=1, N=n, K=64, ldx=64, out=far) == EUNSUP
    assert _grouped(lib, E=1, N=n, K=64, ldx=64, out=far) == EUNSUP
    assert _matmul(lib, M=1, N=2 ** 31 - 257, K=64, ldx=64, out=far) == _lib.QKV_ECUDA


@pytest.mark.parametrize("call,over", [
    # w is 4096 bytes, scales and biases 256 each, of 4 experts four times that; out 256 and 512
    (_matmul, dict(w=(1 << 20) + 240)), (_matmul, dict(w=(1 << 20) - 4080)),
    (_matmul, dict(s=(1 << 20) + 254)), (_matmul, dict(b=(1 << 20) - 254)),
    (_grouped, dict(w=(1 << 20) - 16368)), (_grouped, dict(s=(1 << 20) - 1022)),
    (_grouped, dict(offsets=(1 << 20) - 16)), (_grouped, dict(rows=(1 << 20) + 508)),
    (_combine, dict(slots=(1 << 20) + 508)), (_combine, dict(weights=(1 << 20) - 124)),
    # 2048 x 256 gathered rows: a workspace of 1 MiB
    (_grouped, dict(R=2048, x_rows=2048, rows=1 << 30, out=1 << 29, N=1024, ws=(1 << 29) + 4194288)),
    (_grouped, dict(R=2048, x_rows=2048, rows=1 << 30, out=1 << 29, N=1024, ws=16)),
])
def test_results_apart_from_all_that_is_read(call, over):
    lib = _lib.load()
    assert call(lib, **over) == EINVAL
    assert b"overlaps" in lib.qkv_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch on addresses that are none")
def test_combine_asks_for_vectors_only_where_rows_are_whole_ones():
    lib = _lib.load()
    odd = dict(N=63, y=34, out=(1 << 20) + 2)
    assert _combine(lib, **odd, residual=(1 << 21) + 6) == _lib.QKV_ECUDA
    assert _combine(lib, **(odd | dict(y=33))) == EALIGN
    assert _combine(lib, **(odd | dict(N=64))) == EALIGN
