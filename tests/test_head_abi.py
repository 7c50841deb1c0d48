"""CPU: the lm_head's calls refuse bad arguments with the documented codes before touching the GPU."""


def test_refusals_need_no_gpu():
    from rapid_sampling_b200 import abi
    L = abi.load()

    def quantize(src=4096, dtype=2, V=300, K=256, stride=256, codes=4096, scales=4096):
        return L.rs_head_quantize(src, dtype, V, K, stride, codes, scales, None)
    assert quantize(dtype=3) == abi.RS_ERR_DTYPE
    assert quantize(V=0) == abi.RS_ERR_BATCH
    assert quantize(V=16777217) == quantize(K=0) == quantize(K=250) == quantize(K=65552) == quantize(stride=-1) == abi.RS_ERR_LIMIT
    assert quantize(src=None) == quantize(codes=None) == quantize(scales=None) == abi.RS_ERR_POINTER
    assert quantize(src=4097) == quantize(codes=4104) == quantize(scales=4098) == quantize(src=4098, dtype=0) == abi.RS_ERR_POINTER

    need = L.rs_head_workspace_bytes(5, 256)
    assert need >= 5 * 256 + 2 * 5 * 4 and L.rs_head_workspace_bytes(0, 256) == L.rs_head_workspace_bytes(5, 250) == 0

    def logits(hidden=4096, hdt=2, M=5, K=256, hstride=256, codes=4096, scales=4096, V=300, out=4096, odt=0, ostride=300, ws=4096, n=need):
        return L.rs_head_logits(hidden, hdt, M, K, hstride, codes, scales, V, out, odt, ostride, ws, n, None)
    assert logits(hdt=3) == logits(odt=-1) == abi.RS_ERR_DTYPE
    assert logits(M=0) == logits(V=0) == abi.RS_ERR_BATCH
    assert logits(K=8) == logits(K=65552) == logits(M=16777217) == logits(ostride=299) == logits(hstride=-1) == abi.RS_ERR_LIMIT
    for name in ("hidden", "codes", "scales", "out", "ws"):
        assert logits(**{name: None}) == abi.RS_ERR_POINTER, name
    assert logits(hidden=4097) == logits(codes=4104) == logits(scales=4098) == logits(out=4098) == logits(ws=4224) == abi.RS_ERR_POINTER
    assert logits(n=need - 1) == abi.RS_ERR_WORKSPACE


def test_offered_by_the_package():
    import rapid_sampling_b200 as rs
    assert "lm_head_quantize" in rs.__all__ and "lm_head_logits" in rs.__all__
