"""Refusals of the 4-bit operators and the router of balanced models, before any
launch; runs without a GPU."""
import ctypes

import pytest
import torch

import cvmm_codex_amd as C
from cvmm_codex_amd import _native as N
from oracle import mx4_oracle as O

FAKE = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def lib():
    if not N.available():
        from cvmm_codex_amd import build
        build.build(verbose=False)
    return N.lib()


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        C.cvmm_route_scored(torch.randn(4, 8), 2)
    with pytest.raises(RuntimeError, match="GPU"):
        C.cvmm_mx4_quantize(torch.randn(4, 64))
    keys = C.CVMMMx4(torch.zeros(2, 4096, dtype=torch.uint8), torch.zeros(2, 256, dtype=torch.uint8),
                     torch.Size([2, 64, 64]), 1)
    with pytest.raises(RuntimeError, match="GPU"):
        C.cvmm_mx4(torch.randn(4, 64).bfloat16(), torch.zeros(4, 1, dtype=torch.long), keys)
    with pytest.raises(RuntimeError, match="GPU"):
        keys.dequantize()
    with pytest.raises(TypeError):
        C.cvmm_mx4(torch.randn(4, 64), torch.zeros(4, 1, dtype=torch.long), torch.randn(2, 64, 64))


def test_router_arguments(lib):
    def call(E=16, k=2, scores=1, groups=4, kept=2, dtype=N.F32, ws=None, ws_bytes=0, T=8):
        return lib.cvmm_route_scored(FAKE, dtype, T, E, E, k, None, scores, groups, kept, 1, 1.0, FAKE, FAKE, FAKE,
                                     FAKE, FAKE, FAKE, FAKE, ws, ws_bytes, None)
    assert call(dtype=7) == 1
    assert call(scores=2) == 1 and b"scores" in lib.cvmm_last_error()
    assert call(groups=0) == 1
    assert call(groups=3) == 1                 # 16 experts in 3 groups
    assert call(kept=0) == 1
    assert call(kept=5) == 1
    assert call(k=9) == 1                      # 2 groups of 4 experts stay
    assert call(k=17) == 1
    assert call(E=2048, groups=1, kept=1) == 2
    assert call(E=1024, k=65, groups=1, kept=1) == 2
    assert call(E=512, groups=128, kept=64) == 2
    assert call() == 3 and b"workspace" in lib.cvmm_last_error()
    assert lib.cvmm_route_scored_backward(FAKE, N.F32, 8, 16, 16, 2, 1, 1, 1.0, FAKE, FAKE, FAKE, 8, None) == 1
    assert lib.cvmm_route_scored_backward(FAKE, N.F32, 8, 16, 16, 2, 3, 1, 1.0, FAKE, FAKE, FAKE, 16, None) == 1
    assert lib.cvmm_route_scored_backward(None, N.F32, 8, 16, 16, 2, 1, 1, 1.0, FAKE, FAKE, FAKE, 16, None) == 1
    # counts of every chunk (8 tokens of a short call, 64 of a long one) and the workspace's tail
    need = lib.cvmm_route_scored_workspace_bytes
    assert need(16, 64, 8) >= 65 * 4 and need(32, 256, 8) >= 4 * 257 * 4
    assert need(16384, 128, 8) >= 256 * 129 * 4
    assert need(1 << 20, 1024, 8) <= 3 * 65536 * 4
    assert need(-1, 64, 8) == 0
    # no tokens: nothing to do
    assert lib.cvmm_route_scored_backward(None, N.F32, 0, 16, 16, 2, 1, 1, 1.0, None, None, None, 16, None) == 0


def test_sizes_of_the_layouts(lib):
    assert lib.cvmm_mx4_rows_bytes(3, 32, 0) == 3 * 64 and lib.cvmm_mx4_rows_bytes(3, 32, 1) == 3 * 16
    assert lib.cvmm_mx4_rows_bytes(1, 513, 0) == 320 and lib.cvmm_mx4_rows_bytes(1, 513, 1) == 32
    assert lib.cvmm_mx4_rows_bytes(1, 0, 0) == 0
    assert lib.cvmm_mx4_keys_bytes(2, 128, 64, 0) == 2 * 4096 and lib.cvmm_mx4_keys_bytes(2, 128, 64, 1) == 2 * 256
    assert lib.cvmm_mx4_keys_bytes(1, 129, 65, 0) == 4 * 4096
    assert lib.cvmm_mx4_keys_bytes(130, 8192, 8192, 0) == 130 * 8192 * 8192 // 2
    assert lib.cvmm_mx4_keys_bytes(0, 128, 64, 0) == 0


def test_quantiser_arguments(lib):
    assert lib.cvmm_mx4_quantize_rows(FAKE, 5, 64, 4, 64, FAKE, FAKE, None) == 1
    assert lib.cvmm_mx4_quantize_rows(FAKE, N.F32, 32, 4, 64, FAKE, FAKE, None) == 1      # rows overlap
    assert lib.cvmm_mx4_quantize_rows(FAKE, N.F32, 64, 4, 0, FAKE, FAKE, None) == 1
    assert lib.cvmm_mx4_quantize_rows(None, N.F32, 64, 4, 64, FAKE, FAKE, None) == 1
    assert lib.cvmm_mx4_quantize_rows(None, N.F32, 64, 0, 64, None, None, None) == 0
    assert lib.cvmm_mx4_quantize_keys(FAKE, N.F32, 0, 64, 64, 1, 1, 1, FAKE, FAKE, None) == 1
    assert lib.cvmm_mx4_quantize_keys(FAKE, 9, 2, 64, 64, 1, 1, 1, FAKE, FAKE, None) == 1
    assert lib.cvmm_mx4_quantize_keys(FAKE, N.F32, 2, 64, 64, 1, 1, 1, None, FAKE, None) == 1
    assert lib.cvmm_mx4_dequantize_rows(FAKE, FAKE, 4, 64, FAKE, 4, None) == 1
    assert lib.cvmm_mx4_dequantize_keys(FAKE, FAKE, 2, 64, 0, FAKE, N.F32, None) == 1


def test_product_arguments(lib):
    def fwd(dtype=N.BF16, rows=8, ld=64, E=4, K=64, n=32, R=16, rw=None, k=1, out_rows=16, ws=None, ws_bytes=0,
            quantize=0, x=FAKE):
        return lib.cvmm_mx4_fwd(x, dtype, rows, ld, FAKE, FAKE, E, K, n, FAKE, FAKE, R, FAKE, FAKE, rw, k, quantize,
                                FAKE, out_rows, n, ws, ws_bytes, None)
    assert fwd(dtype=N.F32) == 1 and b"16-bit" in lib.cvmm_last_error()
    assert fwd(E=0) == 1 and fwd(K=0) == 1 and fwd(ld=32) == 1
    assert fwd(out_rows=15) == 1
    assert fwd(rw=FAKE, k=3, out_rows=5) == 1
    assert fwd(rw=FAKE, k=0, out_rows=16) == 1
    assert fwd(rw=FAKE, k=2, out_rows=8) == 3                    # no route buffer
    assert fwd(quantize=1) == 3
    assert fwd(K=60, ld=60) == 3                                 # rows to be copied
    assert fwd(x=None) == 1
    assert fwd(R=0, out_rows=0) == 0

    def bwd(op=N.BF16, rows=16, ld=32, rw=None, k=2, gx=FAKE, gxd=N.BF16, gx_rows=8, grw=None, ws=None, ws_bytes=0,
            oi=FAKE):
        return lib.cvmm_mx4_bwd_x(FAKE, op, rows, ld, FAKE, FAKE, 4, 64, 32, FAKE, oi, 16, FAKE, FAKE, rw, k, FAKE,
                                  N.BF16, 8, 64, gx, gxd, gx_rows, 64, grw, ws, ws_bytes, None)
    assert bwd(op=N.F32) == 1
    assert bwd(gxd=N.F16) == 1
    assert bwd(rows=15) == 1
    assert bwd(ld=16) == 1
    assert bwd(gx_rows=16) == 1
    assert bwd(grw=FAKE) == 1                                    # no routing weights to have a gradient
    assert bwd() == 3                                            # the route buffer of the sum
    assert bwd(gx=None) == 0
    q = lib.cvmm_mx4_bwd_x_workspace_bytes
    assert q(16, 64, 32, 16, 1, 1, 0, 0, N.BF16) == 16 * 64 * 2
    assert q(16, 64, 32, 16, 0, 1, 0, 0, N.BF16) == 0
    f = lib.cvmm_mx4_fwd_workspace_bytes
    assert f(16, 64, 32, 8, 0, 1, 0, 0) == 0 and f(16, 64, 32, 8, 1, 1, 0, 0) == 16 * 32 * 2


def test_oracle_quantises_by_the_definition():
    v = torch.tensor([[4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -5.0, 0.3, -0.2]])
    assert O.quantize(v).tolist() == [[4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, -4.0, 0.5, -0.0]]
    assert torch.equal(O.quantize(v * 2.0 ** -100), O.quantize(v) * 2.0 ** -100)
    w = torch.randn(2, 70, 3)
    assert torch.equal(O.quantize(w, 1), O.quantize(w.transpose(1, 2)).transpose(1, 2))


def test_oracle_routes_within_the_best_groups():
    logits = torch.tensor([[3.0, -5.0, 1.0, 1.5, 0.0, 0.0, 2.9, -9.0]])
    w, sel = O.route(logits, 2, scores="sigmoid", groups=4, topk_groups=1)
    assert sel.tolist() == [[3, 2]]            # the pair (1, 1.5) beats (3, -5)
    assert abs(float(w.sum()) - 1) < 1e-12


def test_buffers_have_to_fit_the_shape(lib):
    """What a caller puts together from stored codes and scales is checked before
    any kernel reads them by the shape."""
    def buf(n, at=0):
        return torch.zeros(n + 64, dtype=torch.uint8)[at:at + n]

    check = N.host().mx4_check
    for shape, keys, codes, scales in (([2, 128, 64], True, 2 * 4096, 2 * 256), ([1, 129, 65], True, 4 * 4096, 4 * 256),
                                       ([3, 200], False, 3 * 128, 3 * 16), ([2, 3, 513], False, 6 * 320, 6 * 32),
                                       ([0, 64], False, 0, 0)):
        assert check(buf(codes), buf(scales), shape, keys, "t") is None
        bad = [(buf(codes + 16), buf(scales)), (buf(codes), buf(scales + 4)), (buf(codes).char(), buf(scales)),
               (buf(codes), buf(scales).char())]
        if codes:
            bad += [(buf(codes - 16), buf(scales)), (buf(codes), buf(scales - 4)), (buf(codes, 2), buf(scales)),
                    (torch.zeros(2 * codes, dtype=torch.uint8)[::2], buf(scales)),
                    (buf(codes), torch.zeros(2 * scales, dtype=torch.uint8)[::2])]
        if keys:
            bad += [(buf(codes, 4), buf(scales)), (buf(codes), buf(scales, 1))]
        for c, s in bad:
            with pytest.raises(ValueError, match="shape"):
                check(c, s, shape, keys, "t")
        if codes:  # a larger or an impossible shape
            for other in ([*shape[:-1], shape[-1] + 512], [*shape[:-1], 0], [-1, *shape[1:]], [shape[0] + 1, *shape[1:]]):
                with pytest.raises(ValueError, match="shape"):
                    check(buf(codes), buf(scales), other, keys, "t")
    for shape in ([64], [2, 64], [2, 2, 64, 64]):
        with pytest.raises(ValueError, match="shape"):
            check(buf(8192), buf(512), shape, True, "t")
    with pytest.raises(ValueError, match="shape"):
        check(buf(0), buf(0), [], False, "t")


def test_dims_of_a_4_bit_tensor():
    def make(shape, dim):
        return C.CVMMMx4(torch.zeros(1, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8), torch.Size(shape), dim)
    assert make([2, 128, 128], -1).dim == 2 and not make([2, 128, 128], -1)._keys
    assert make([2, 128, 128], -2).dim == 1 and make([2, 128, 128], 1)._keys
    assert not make([4, 64], 1)._keys and not make([64], 0)._keys
    for shape, dim in (([2, 64, 64], 0), ([2, 64], 0), ([2, 64], 2), ([2, 64], -3), ([2, 3, 64, 64], 1), ([], 0)):
        with pytest.raises(ValueError, match="dim"):
            make(shape, dim)


def test_row_indices_fit_32_bits(lib):
    """The products hold row indices in 32 bits: more rows are refused, not read as
    none."""
    def fwd(rows):
        return lib.cvmm_mx4_fwd(FAKE, N.BF16, rows, 64, FAKE, FAKE, 4, 64, 32, FAKE, FAKE, 16, FAKE, FAKE, None, 1, 0,
                                FAKE, 16, 32, None, 0, None)
    assert fwd(2 ** 31) == 1 and b"sizes" in lib.cvmm_last_error()
