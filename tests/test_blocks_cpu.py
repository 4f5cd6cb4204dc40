"""What of the 8-bit block operators and the token log probabilities needs no GPU: the checks of arguments on the
host side, and the tests' own definitions against a second source."""
import numpy as np
import pytest
import torch

from gorgonia_b200 import B200Error, BlockTensor, Engine, Tensor, _lib
from gorgonia_b200._lib import lib
from tests import blocks_util as bu


@pytest.fixture()
def e():
    """An engine without a device: its checks run, and the library refuses the null handle behind them."""
    x = Engine.__new__(Engine)
    x.h = None
    return x


def tensor(e, shape, dtype=np.float32, bf16=False):
    shape = (shape,) if isinstance(shape, int) else shape
    t = Tensor(e, 4096, shape, np.uint16 if bf16 else dtype, owned=False)
    if bf16:
        t.is_bf16 = True
    return t


def blocks(e, shape, fmt="e4m3", block="row"):
    return BlockTensor(tensor(e, shape, np.uint8), tensor(e, BlockTensor.scale_shape(shape, block)), fmt, block)


def refused(call, *args, text, code=_lib.ERR_INVALID, **kw):
    with pytest.raises(B200Error, match=text) as err:
        call(*args, **kw)
    assert err.value.code == code


@pytest.mark.parametrize("fmt,dt", [("e4m3", torch.float8_e4m3fn), ("e5m2", torch.float8_e5m2)])
def test_definition_of_the_formats(fmt, dt):
    v = bu.f8_values(fmt)
    t = torch.arange(256, dtype=torch.uint8).view(dt).to(torch.float64).numpy()
    assert np.array_equal(v, t, equal_nan=True)
    x = np.random.default_rng(3).standard_normal((7, 300)).astype(np.float32)
    q, s = bu.quantize(x, fmt, "row")
    again = torch.from_numpy((x / bu.spread(s, x.shape, "row")).astype(np.float32)).to(dt).to(torch.float64).numpy()
    assert np.array_equal(q, again)
    assert np.array_equal(bu.f8_values(fmt)[bu.to_bytes(q, fmt)], q)


def test_definition_of_log_probabilities():
    x = np.random.default_rng(4).standard_normal((5, 40))
    x[1, :30] = -np.inf
    t = np.array([0, 35, 39, -1, 7])
    d = bu.logprobs(x, t, 3)
    xt = torch.from_numpy(x).requires_grad_()
    lp = torch.log_softmax(xt, 1)
    p = lp.exp()
    ent = torch.distributions.Categorical(logits=xt).entropy()
    assert np.allclose(d["lse"], torch.logsumexp(xt, 1).detach().numpy())
    assert np.allclose(d["entropy"][[0, 2, 3, 4]], ent.detach().numpy()[[0, 2, 3, 4]])
    some = (-p * lp).nan_to_num(0.0).sum(1)
    assert np.allclose(d["entropy"], some.detach().numpy())
    assert np.allclose(d["top_logp"], torch.topk(lp, 3, 1).values.detach().numpy())
    g, h = np.array([1.0, 0.5, -2, 3, 0.25]), np.array([0.1, 0, -0.3, 0, 2.0])
    on = torch.from_numpy(t >= 0)
    logp = lp.gather(1, torch.from_numpy(np.maximum(t, 0))[:, None])[:, 0][on]
    keep = torch.from_numpy(h != 0)
    ((logp * torch.from_numpy(g)[on]).sum() + (ent[keep] * torch.from_numpy(h)[keep]).sum()).backward()
    want = xt.grad.nan_to_num(0.0).numpy()
    got = bu.logprobs_diff(x, t, d["lse"], d["entropy"], g, h)
    assert np.allclose(got, want)


def test_block_tensor_refuses(e):
    q = tensor(e, (200, 300), np.uint8)
    refused(BlockTensor, q, tensor(e, (200, 3)), "e3m4", "row", text="format")
    refused(BlockTensor, q, tensor(e, (200, 3)), "e4m3", "diagonal", text="block")
    refused(BlockTensor, q, tensor(e, (200, 2)), "e4m3", "row", text="scales of shape")
    refused(BlockTensor, q, tensor(e, (200, 3)), "e4m3", "tile", text="scales of shape")
    refused(BlockTensor, q, tensor(e, (200, 3), np.float64), "e4m3", "row", text="float32 scales")
    refused(BlockTensor, tensor(e, (200, 300)), tensor(e, (200, 3)), text="uint8")
    refused(BlockTensor, tensor(e, (2, 100, 300), np.uint8), tensor(e, (200, 3)), text="matrix")
    assert [BlockTensor.scale_shape((129, 128), b) for b in ("row", "col", "tile")] == [(129, 1), (2, 128), (2, 1)]


def test_quantize_refuses(e):
    refused(e.QuantizeBlocks, tensor(e, (4, 128)), blocks(e, (4, 127)), text="does not fit")
    refused(e.QuantizeBlocks, tensor(e, (4, 128), np.int64), blocks(e, (4, 128)), text="not supported", code=_lib.ERR_UNSUPPORTED)


def test_matmul_refuses(e):
    a, b = blocks(e, (64, 256)), blocks(e, (32, 256), block="tile")
    c = tensor(e, (64, 32))
    refused(e.MatMulBlocks, a, b, c, text="inner dimensions")
    refused(e.MatMulBlocks, a, b, tensor(e, (64, 31)), transB=True, text="wrong size")
    refused(e.MatMulBlocks, a, b, c, transB=True, bias=tensor(e, 31), text="bias")
    refused(e.MatMulBlocks, a, b, c, transB=True, bias=tensor(e, 32), bias_kind="row", text="bias")
    refused(e.MatMulBlocks, a, b, c, transB=True, bias=tensor(e, 32, np.float64), text="bias")


def test_logprobs_refuse(e):
    x, t = tensor(e, (6, 50)), tensor(e, 6, np.int64)
    refused(e.TokenLogProbs, x, t, tensor(e, 5), text="logp has to hold")
    refused(e.TokenLogProbs, x, t, tensor(e, 6, np.float64), text="logp has to hold")
    refused(e.TokenLogProbs, x, tensor(e, 6, np.int32), tensor(e, 6), text="int64")
    refused(e.TokenLogProbs, x, tensor(e, 7, np.int64), tensor(e, 6), text="int64")
    refused(e.TokenLogProbs, x, t, tensor(e, 6), top_logp=tensor(e, (6, 2)), top_index=tensor(e, (6, 3), np.int64), text="top_logp")
    refused(e.TokenLogProbs, x, t, tensor(e, 6), top_logp=tensor(e, 13), top_index=tensor(e, 13, np.int64), text="top_logp")
    d = tensor(e, (6, 50), np.float64)
    refused(e.TokenLogProbs, d, t, tensor(e, 6), text="logp has to hold")
    s = tensor(e, 6)
    refused(e.TokenLogProbsDiff, x, t, s, s, s, tensor(e, (6, 49)), text="prealloc")
    refused(e.TokenLogProbsDiff, x, t, s, s, s, tensor(e, (6, 50), bf16=True), text="prealloc")
    refused(e.TokenLogProbsDiff, x, t, s, s, tensor(e, 5), x, text="grad_logp")
    refused(e.TokenLogProbsDiff, x, tensor(e, 5, np.int64), s, s, s, x, text="targets")


def test_null_engine_is_refused():
    assert lib.b200_quantize_blocks(None, 0, 3, 0, None, 0, 0, 0, None, 0, None) == _lib.ERR_INVALID
    assert lib.b200_gemm_blocks(None, 0, 0, 0, 0, 0, 0, None, 3, 0, 0, None, None, 3, 2, 0, None, None, 0, None) == _lib.ERR_INVALID
    assert lib.b200_token_logprobs(None, 0, None, 0, 0, 1, None, None, None, None, 0, None, None) == _lib.ERR_INVALID
    assert lib.b200_token_logprobs_bwd(None, 0, None, 0, 0, 1, None, None, None, None, None, None, 0) == _lib.ERR_INVALID
