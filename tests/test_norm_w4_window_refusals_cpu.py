"""What K6, K7 and K8 refuse. Arguments are checked before any CUDA call, so no GPU is needed; the addresses are never read."""
import pytest

from cubert_b200 import kernels

A = 0x10000                                    # an aligned address that nothing dereferences
INVALID, UNSUPPORTED = kernels.CUBK_ERR_INVALID_ARG, kernels.CUBK_ERR_UNSUPPORTED
NAN = float("nan")


def refused(name, good, changes):
    """`good` with one or more arguments replaced at a time returns the status given with the change."""
    for at, value, status in changes:
        args = list(good)
        for i, v in zip(at if isinstance(at, tuple) else (at,), value if isinstance(at, tuple) else (value,)):
            args[i] = v
        for t in ("f32", "f16"):
            assert getattr(kernels.load(), "cubk_%s_%s" % (name, t))(*args) == status, (name, t, at, value)


def test_rms_norm():
    good = (A, A, A, 4, 64, 1e-6, A, A, None)      # x, residual, gamma, rows, channels, eps, sum, out, stream
    refused("residual_rms_norm", good, [(0, None, INVALID), (2, None, INVALID), (7, None, INVALID), (3, -1, INVALID), (4, 0, INVALID),
                                        (4, -8, INVALID), (5, -1.0, INVALID), (5, NAN, INVALID), (3, 0, 0)])
    good = (A, A, A, 4, 64, 1e-6, 0, A, A, A, None)   # ..., eps, group, sum, codes, scales, stream
    refused("residual_rms_norm_e4m3", good, [(0, None, INVALID), (2, None, INVALID), (8, None, INVALID), (9, None, INVALID), (3, -1, INVALID),
                                             (4, 0, INVALID), (6, 64, INVALID), (6, -1, INVALID), (3, 0, 0)])


def test_w4_matvec():
    good = (A, 2, 256, A, A, 64, 32, A, A, None)   # x, rows, k, packed, scales, group, n, bias, out, stream
    refused("w4_matvec", good, [(0, None, INVALID), (3, None, INVALID), (4, None, INVALID), (8, None, INVALID), (1, -1, INVALID), (2, 0, INVALID),
                                (6, 0, INVALID), (5, 0, INVALID), (5, 48, INVALID), (5, 256, INVALID), (3, A + 8, UNSUPPORTED), (4, A + 2, UNSUPPORTED), (2, 2 ** 30 + 1, UNSUPPORTED),
                                (6, 2 ** 30 + 1, UNSUPPORTED), (1, 16 * 65535 + 1, UNSUPPORTED), (1, 0, 0)])
    good = (A, A, 0, 2, 256, A, A, 64, 32, A, A, None)   # codes, code_scales, code_group, rows, ...
    refused("w4_matvec_e4m3", good, [(0, None, INVALID), (1, None, INVALID), (2, 64, INVALID), (3, -1, INVALID), (5, None, INVALID),
                                     (6, None, INVALID), (10, None, INVALID), (5, A + 4, UNSUPPORTED), (7, 16, INVALID), (3, 0, 0)])


def test_w4_layout():
    good = (A, 16, 256, 64, A, A, None)            # weights, n, k, group, packed, scales, stream
    refused("w4_quantize", good, [(0, None, INVALID), (4, None, INVALID), (5, None, INVALID), (1, 0, INVALID), (2, 0, INVALID), (3, 100, INVALID),
                                  (4, A + 1, UNSUPPORTED)])
    lib = kernels.load()
    assert lib.cubk_w4_pack(None, 16, 256, A, None) == INVALID
    assert lib.cubk_w4_pack(A, 0, 256, A, None) == INVALID
    assert lib.cubk_w4_pack(A, 16, 256, A + 2, None) == UNSUPPORTED
    assert lib.cubk_w4_packed_bytes(0, 4) == 0 and lib.cubk_w4_packed_bytes(4, -1) == 0
    assert lib.cubk_w4_packed_bytes(1, 1) == 1024 and lib.cubk_w4_packed_bytes(17, 129) == 4096
    assert lib.cubk_w4_packed_bytes(2 ** 31 - 1, 2 ** 31 - 1) == 2 ** 27 * 2 ** 24 * 1024


def test_window_attention():
    # q, k, v, q_stride, kv_stride, mask, batch, seq, heads, kv_heads, dim, before, after, sinks, scale, context, context_stride, stream
    good = (A, A, A, 512, 512, A, 2, 10, 8, 2, 64, 3, 0, 1, 0.125, A, 512, None)
    refused("window_attention", good, [(0, None, INVALID), (1, None, INVALID), (2, None, INVALID), (15, None, INVALID), (3, 511, INVALID),
                                       (4, 127, INVALID), (16, 500, INVALID), (6, -1, INVALID), (7, -1, INVALID), (8, 0, INVALID), (9, 3, INVALID),
                                       (9, 0, INVALID), (10, 0, INVALID), (11, -1, INVALID), (12, -1, INVALID), (13, -1, INVALID),
                                       ((10, 3, 4, 16), (257, 4096, 4096, 4096), UNSUPPORTED), (7, 2 ** 30, UNSUPPORTED), (6, 0, 0), (7, 0, 0)])


def test_window_attention_step():
    # q, k, v, q_stride, kv_stride, positions, batch, heads, kv_heads, dim, window, sinks, scale, k_cache, v_cache, context, context_stride, stream
    good = (A, A, A, 512, 512, A, 2, 8, 2, 64, 10, 1, 0.125, A, A, A, 512, None)
    refused("window_attention_step", good, [(0, None, INVALID), (1, None, INVALID), (2, None, INVALID), (5, None, INVALID), (13, None, INVALID),
                                            (14, None, INVALID), (15, None, INVALID), (3, 511, INVALID), (4, 127, INVALID), (16, 500, INVALID),
                                            (6, -1, INVALID), (7, 0, INVALID), (8, 3, INVALID), (9, 0, INVALID), (10, 0, INVALID), (11, -1, INVALID),
                                            ((9, 3, 4, 16), (257, 4096, 4096, 4096), UNSUPPORTED), (10, 2 ** 30, UNSUPPORTED), (6, 0, 0)])


def test_window_cache_fill():
    # k, v, kv_stride, lengths, batch, seq, kv_heads, dim, window, sinks, k_cache, v_cache, stream
    good = (A, A, 128, A, 2, 10, 2, 64, 10, 1, A, A, None)
    refused("window_cache_fill", good, [(0, None, INVALID), (1, None, INVALID), (10, None, INVALID), (11, None, INVALID), (2, 127, INVALID),
                                        (4, -1, INVALID), (5, -1, INVALID), (6, 0, INVALID), (7, 0, INVALID), (8, 0, INVALID), (9, -1, INVALID),
                                        ((7, 2), (257, 1024), UNSUPPORTED), (8, 2 ** 30, UNSUPPORTED), (9, 2 ** 30, UNSUPPORTED), (4, 0, 0), (5, 0, 0)])


def test_every_entry_point_is_bound():
    names = kernels.exported_symbols()
    for stem in ("residual_rms_norm", "residual_rms_norm_e4m3", "w4_quantize", "w4_matvec", "w4_matvec_e4m3", "window_attention",
                 "window_attention_step", "window_cache_fill"):
        assert {"cubk_%s_f32" % stem, "cubk_%s_f16" % stem} <= set(names)
    with pytest.raises(kernels.KernelError):
        kernels.check(kernels.load().cubk_w4_pack(None, 1, 1, None, None))
