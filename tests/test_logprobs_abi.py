"""CPU: the log probability calls refuse bad arguments with the documented codes before touching the GPU."""
import ctypes as C


def _call(abi, **kw):
    c = abi.LogprobCall()
    c.logits = c.tokens = 4096
    c.B, c.T, c.V, c.stride_b, c.stride_t = 2, 3, 1000, 3000, 1000
    c.temperature, c.dtype, c.token_bits = 1.0, abi.RS_DTYPE_F32, 64
    for k, v in kw.items():
        setattr(c, k, v)
    return C.byref(c)


BAD = [(dict(V=0), "RS_ERR_LIMIT"), (dict(V=1048577), "RS_ERR_LIMIT"), (dict(B=0), "RS_ERR_BATCH"), (dict(T=0), "RS_ERR_BATCH"),
       (dict(T=-1), "RS_ERR_BATCH"), (dict(B=1 << 20, T=1 << 20), "RS_ERR_LIMIT"), (dict(T=1 << 31), "RS_ERR_LIMIT"),
       (dict(temperature=0.0), "RS_ERR_TEMPERATURE"), (dict(temperature=1001.0), "RS_ERR_TEMPERATURE"),
       (dict(temperature=float("nan")), "RS_ERR_TEMPERATURE"), (dict(logits=None), "RS_ERR_POINTER"), (dict(logits=4098), "RS_ERR_POINTER"),
       (dict(logits=4097, dtype=1), "RS_ERR_POINTER"), (dict(tokens=4100), "RS_ERR_POINTER"), (dict(tokens=4098, token_bits=32), "RS_ERR_POINTER"),
       (dict(dtype=3), "RS_ERR_DTYPE"), (dict(token_bits=16), "RS_ERR_DTYPE"), (dict(row_temperature=4098), "RS_ERR_POINTER")]


def test_refusals_need_no_gpu():
    from rapid_sampling_b200 import abi
    L = abi.load()
    for kw, code in BAD:
        want = getattr(abi, code)
        assert L.rs_token_logprobs(_call(abi, **kw), 4096, 4096, 4096) == want, kw
        assert L.rs_token_logprobs_backward(_call(abi, **kw), 4096, 4096, 4096, 3, 1, 4096, 3, 1, 4096) == want, kw
        assert L.rs_top_logprobs(_call(abi, **kw), 5, 4096, 4096, 4096, 4096, 4096) == want, kw
    assert L.rs_token_logprobs(None, 4096, 4096, None) == abi.RS_ERR_POINTER
    assert L.rs_top_logprobs(None, 5, 4096, 4096, 4096, 4096, 4096) == abi.RS_ERR_POINTER
    assert L.rs_token_logprobs(_call(abi, tokens=None), 4096, 4096, None) == abi.RS_ERR_POINTER


def test_offered_by_the_package():
    import rapid_sampling_b200 as rs
    assert "batch_token_logprobs" in rs.__all__ and "batch_top_logprobs" in rs.__all__
    from rapid_sampling_b200 import abi
    assert abi.status_string(abi.RS_ERR_TOKEN) == "a token id is no column of the logits"


def test_forward_mode_is_refused():
    import pytest
    import torch
    import torch.autograd.forward_ad as fwd
    import rapid_sampling_b200 as rs
    x, t = torch.zeros(2, 5), torch.zeros(2, dtype=torch.long)
    with fwd.dual_level():
        with pytest.raises(ValueError, match="tangents"):
            rs.batch_token_logprobs(fwd.make_dual(x, torch.ones_like(x)), t)
        with pytest.raises(ValueError, match="CUDA"):
            rs.batch_token_logprobs(x, t)
    with pytest.raises(ValueError, match="tangents"):
        torch.func.jvp(lambda y: rs.batch_token_logprobs(y, t)[0], (x,), (torch.ones_like(x),))
