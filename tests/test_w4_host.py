"""Argument checks of the 4-bit weights' entry points: host code, no GPU."""

import ctypes

import pytest
import torch

from wkvm_amd import W4Weight, _lib, proj_w4

A, S, OK = _lib.WKV7_ERR_ARG, _lib.WKV7_ERR_SHAPE, _lib.WKV7_OK
P = ctypes.c_void_p(4096)


def _desc(**kw):
    d = _lib.W4Desc(4096, 4096, 48, 64, 32, 0)
    for name, value in kw.items():
        setattr(d, name, value)
    return d


WEIGHTS = [(dict(codes=None), A), (dict(scales=None), A), (dict(n=0), A), (dict(k=0), A),
           (dict(k=48), A), (dict(group=16), A), (dict(group=0), A), (dict(codes=4104), S),
           (dict(scales=4100), S)]


@pytest.mark.parametrize("change,code", WEIGHTS)
def test_abi_refuses_weights(change, code):
    lib, d = _lib.load(), _desc(**change)
    assert lib.wkv7_w4_pack(d, P, P, 0, None, None) == code
    assert lib.wkv7_w4_quantize(d, P, 64, 0, None) == code
    assert lib.wkv7_w4_unpack(d, P, None) == code
    groups = (_lib.W4Group * 1)(_lib.W4Group(4096, d, None, 4096, 64, 48, 0, 0))
    assert lib.wkv7_proj_w4(2, groups, 1, None, 0, None) == code


@pytest.mark.parametrize("change,code", [
    (dict(x=None), A), (dict(y=None), A), (dict(act=5), A), (dict(ldx=56), S), (dict(ldx=68), S),
    (dict(ldy=47), S), (dict(x=4104), S)])
def test_abi_refuses_products(change, code):
    group = _lib.W4Group(4096, _desc(), None, 4096, 64, 48, 0, 0)
    for name, value in change.items():
        setattr(group, name, value)
    groups = (_lib.W4Group * 2)(_lib.W4Group(4096, _desc(), None, 4096, 64, 48, 0, 0), group)
    assert _lib.load().wkv7_proj_w4(2, groups, 2, None, 0, None) == code


def test_abi_refuses_calls():
    lib = _lib.load()
    groups = (_lib.W4Group * 9)(*[_lib.W4Group(4096, _desc(), None, 4096, 64, 48, 0, 0)] * 9)
    assert lib.wkv7_proj_w4(-1, groups, 1, None, 0, None) == A
    assert lib.wkv7_proj_w4(1 << 31, groups, 1, None, 0, None) == A
    assert lib.wkv7_proj_w4(1, groups, 0, None, 0, None) == A
    assert lib.wkv7_proj_w4(1, groups, 9, None, 0, None) == A
    assert lib.wkv7_proj_w4(1, None, 1, None, 0, None) == A
    assert lib.wkv7_proj_w4(0, groups, 1, None, 0, None) == OK
    assert lib.wkv7_proj_w4_workspace_bytes(64, groups, 8) == 0
    need = lib.wkv7_proj_w4_workspace_bytes(65, groups, 2)
    assert need == 2 * 96 * 3 * 16 * 2  # three bf16 parts of 16 groups' sums (two there), rows by 32
    assert lib.wkv7_proj_w4(65, groups, 2, None, need, None) == _lib.WKV7_ERR_WORKSPACE
    assert lib.wkv7_proj_w4(65, groups, 2, P, need - 1, None) == _lib.WKV7_ERR_WORKSPACE
    assert lib.wkv7_proj_w4(65, groups, 2, ctypes.c_void_p(4104), need, None) == S
    d = _desc()
    assert lib.wkv7_w4_pack(d, None, P, 0, None, None) == A
    assert lib.wkv7_w4_pack(d, P, None, 0, None, None) == A
    assert lib.wkv7_w4_pack(d, P, P, 2, None, None) == A
    assert lib.wkv7_w4_pack(d, P, ctypes.c_void_p(4097), 0, None, None) == S
    assert lib.wkv7_w4_quantize(d, None, 64, 0, None) == A
    assert lib.wkv7_w4_quantize(d, P, 63, 0, None) == S
    assert lib.wkv7_w4_unpack(d, None, None) == A
    assert lib.wkv7_w4_unpack(d, ctypes.c_void_p(4098), None) == S


@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (16, 128, 128), (17, 160, 64), (65536, 2048, 128)])
def test_sizes(n, k, group):
    lib = _lib.load()
    tiles = -(-n // 16)
    assert lib.wkv7_w4_code_bytes(n, k) == tiles * -(-k // 128) * 1024
    assert lib.wkv7_w4_scale_bytes(n, k, group) == tiles * -(-k // group) * 64


def test_python_refusals():
    for args, match in (((0, 64), "n must"), ((4, 48), "multiple of 32"), ((4, 64, 16), "group"),
                        ((4, 0), "multiple of 32")):
        with pytest.raises(ValueError, match=match):
            W4Weight(*args, device="cpu")
    with pytest.raises(ValueError, match="GPU tensor"):
        W4Weight.quantize(torch.zeros(4, 32, dtype=torch.bfloat16))
    weight = W4Weight(4, 32, 32, device="cpu")
    assert weight.shape == (4, 32) and weight.nbytes() == 1024 + 64
    with pytest.raises(ValueError, match="GPU tensor"):
        proj_w4([(torch.zeros(1, 32, dtype=torch.bfloat16), weight)])


def test_block_refuses_other_projections_and_host_weights():
    from wkvm_amd.layout import RWKV7StateLayout
    from wkvm_amd.timemix import RWKV7TimeMix

    block = RWKV7TimeMix.random(RWKV7StateLayout(1, 64, 1, 64, 64, torch.bfloat16), 0, "cpu")
    for names in (("w1",), ("r", "mix"), ("r", "r2")):
        with pytest.raises(ValueError, match="can be 4-bit weights"):
            block.quantize(32, names)
    with pytest.raises(ValueError):  # (on the host)
        block.quantize(32)
    assert not block.w4 and "r" in block.w
    block.add_adapters(2, 8, ("k",))
    with pytest.raises(ValueError, match="holds adapters"):
        block.quantize(32, ("r", "k"))
    block.w4["v"] = object()
    with pytest.raises(ValueError, match="takes no adapters"):
        block.add_adapters(2, 8, ("o", "v"))
    with pytest.raises(ValueError, match="already holds a 4-bit"):
        block.quantize(32, ("v",))
    assert set(block.adapters) == {"k"}


def test_a_host_weight_has_no_values():
    """Its buffers are host memory, which no kernel may be given."""
    with pytest.raises(ValueError, match="GPU tensor"):
        W4Weight(4, 32, 32, device="cpu").dequantize()


def test_a_weight_keeps_its_buffers():
    """The launches hold their addresses: another tensor in their place would not be read, and they
    would be freed. Until they are filled the weight is zero."""
    weight = W4Weight(40, 96, 32, device="cpu")
    for name in ("codes", "scales"):
        with pytest.raises(AttributeError):
            setattr(weight, name, torch.zeros_like(getattr(weight, name)))
        assert not getattr(weight, name).any()
    assert weight.fields[:2] == (weight.codes.data_ptr(), weight.scales.data_ptr())
