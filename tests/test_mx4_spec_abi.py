"""CPU checks of the sampled verification's and the 4-bit floating-point calls'
C ABI and Python front ends: sizes of workspaces and layouts, and bad arguments
refused before any HIP call."""
import ctypes

import pytest
import torch

from hi_amd import _lib, mx4
from hi_amd.speculative import SpecVerifier
from oracle import mx4_oracle, spec_sampled_oracle

ARGS, UNSUPPORTED = _lib.ERR_ARGS, _lib.ERR_UNSUPPORTED
F32, BF16, MX4 = _lib.DTYPE_F32, _lib.DTYPE_BF16, _lib.DTYPE_MX4
P = 1 << 32  # an address on 16 bytes that nothing may touch
BIG = 1 << 40

GOOD = {
    "hi_rocm_spec_verify_sampled": dict(
        target=P, dtype=F32, batch=2, max_draft=3, vocab=1000, target_batch=4000, target_row=1000, draft=P,
        draft_batch=3000, draft_row=1000, tokens=P, lengths=0, uniforms=P, out_tokens=P, out_count=P, workspace=P,
        workspace_bytes=BIG, stream=None),
    "hi_rocm_mx4_quantize": dict(x=P, dtype=BF16, rows=3, k=64, x_stride=64, codes=P, scales=P, stream=None),
    "hi_rocm_mx4_dequantize": dict(codes=P, scales=P, rows=3, k=64, out=P, out_dtype=F32, out_stride=64, stream=None),
    "hi_rocm_mx4_rows": dict(x=P, dtype=BF16, rows=3, k=64, x_stride=64, out=P, out_bytes=BIG, stream=None),
    "hi_rocm_mx4_moe_prepare": dict(
        ids=P, tokens=20, top_k=2, experts=4, order=P, slots=P, offsets=P, x=P, k=64, x_stride=64, out=P, out_bytes=BIG,
        stream=None),
    "hi_rocm_mx4_pack": dict(codes=P, scales=P, experts=2, n=48, k=64, packed=P, packed_bytes=BIG, stream=None),
    "hi_rocm_mx4_linear": dict(
        x=P, x_dtype=BF16, rows=20, x_stride=64, packed=P, packed_bytes=BIG, n=48, k=64, bias=0, out=P, out_dtype=F32,
        out_stride=48, workspace=P, workspace_bytes=BIG, stream=None),
    "hi_rocm_mx4_grouped_product": dict(
        x=P, x_dtype=BF16, x_rows=20, x_stride=64, order=P, top_k=2, offsets=P, places=40, experts=4, packed=P,
        packed_bytes=BIG, cols=128, k=64, swiglu=1, out=P, out_dtype=BF16, out_stride=64, out_bytes=BIG, workspace=P,
        workspace_bytes=BIG, stream=None),
}

REFUSED = [
    ("hi_rocm_spec_verify_sampled", ARGS, [
        dict(target=None), dict(uniforms=None), dict(tokens=None), dict(out_tokens=None), dict(out_count=None),
        dict(workspace=None), dict(workspace=P + 8), dict(workspace_bytes=100), dict(batch=0), dict(batch=-1),
        dict(vocab=0), dict(max_draft=-1), dict(dtype=MX4), dict(target=P + 2), dict(draft=P + 1, dtype=BF16),
        dict(target_row=-1), dict(target_batch=-1), dict(draft_row=-1), dict(draft_batch=-1)]),
    ("hi_rocm_spec_verify_sampled", UNSUPPORTED, [
        dict(batch=65536), dict(vocab=(1 << 23) + 1), dict(max_draft=65536), dict(batch=65535, vocab=1 << 23)]),
    ("hi_rocm_mx4_quantize", ARGS, [
        dict(x=None), dict(codes=None), dict(scales=None), dict(rows=0), dict(k=0), dict(k=-32), dict(dtype=MX4),
        dict(x_stride=63)]),
    ("hi_rocm_mx4_quantize", UNSUPPORTED, [
        dict(k=48), dict(x=P + 8), dict(codes=P + 8), dict(x_stride=68), dict(k=(1 << 24) + 32, x_stride=1 << 25),
        dict(rows=1 << 60), dict(rows=1 << 29)]),
    ("hi_rocm_mx4_dequantize", ARGS, [
        dict(codes=None), dict(scales=None), dict(out=None), dict(rows=-1), dict(k=0), dict(out_dtype=7),
        dict(out_stride=32)]),
    ("hi_rocm_mx4_dequantize", UNSUPPORTED, [
        dict(k=80, out_stride=96), dict(out=P + 8), dict(codes=P + 4), dict(out_stride=66), dict(rows=1 << 29)]),
    ("hi_rocm_mx4_rows", ARGS, [
        dict(x=None), dict(out=None), dict(rows=0), dict(dtype=5), dict(x_stride=32), dict(out=P + 8), dict(out_bytes=64)]),
    ("hi_rocm_mx4_rows", UNSUPPORTED, [dict(k=40), dict(x=P + 2), dict(x_stride=65), dict(rows=1 << 29)]),
    ("hi_rocm_mx4_moe_prepare", ARGS, [
        dict(ids=None), dict(order=None), dict(slots=None), dict(offsets=None), dict(x=None), dict(out=None),
        dict(tokens=0), dict(top_k=0), dict(experts=0), dict(k=0), dict(x_stride=63), dict(out=P + 8),
        dict(out_bytes=100)]),
    ("hi_rocm_mx4_moe_prepare", UNSUPPORTED, [
        dict(experts=2049), dict(tokens=(1 << 21) + 1), dict(k=48), dict(x=P + 8), dict(x_stride=68),
        dict(k=(1 << 24) + 32, x_stride=1 << 25)]),
    ("hi_rocm_mx4_pack", ARGS, [
        dict(codes=None), dict(scales=None), dict(packed=None), dict(experts=0), dict(n=0), dict(k=0), dict(packed=P + 8),
        dict(packed_bytes=1000)]),
    ("hi_rocm_mx4_pack", UNSUPPORTED, [
        dict(k=72), dict(codes=P + 8), dict(experts=2049), dict(n=(1 << 24) + 1), dict(k=1 << 25),
        dict(experts=2048, n=1 << 20, k=1 << 20)]),
    ("hi_rocm_mx4_linear", ARGS, [
        dict(x=None), dict(packed=None), dict(out=None), dict(rows=0), dict(n=0), dict(k=0), dict(x_dtype=F32),
        dict(x_stride=32), dict(out_dtype=MX4), dict(out_stride=47), dict(out=P + 2), dict(out=P + 1, out_dtype=BF16),
        dict(bias=P + 2), dict(packed=P + 8), dict(packed_bytes=100), dict(k=4128, x_stride=4128, workspace=None),
        dict(k=4128, x_stride=4128, workspace=P + 8), dict(k=4128, x_stride=4128, workspace_bytes=100)]),
    ("hi_rocm_mx4_linear", UNSUPPORTED, [
        dict(k=48), dict(rows=(1 << 22) + 1), dict(x=P + 8), dict(x_stride=68), dict(n=(1 << 24) + 1, out_stride=1 << 25),
        dict(x=P + 8, x_dtype=MX4)]),
    ("hi_rocm_mx4_grouped_product", ARGS, [
        dict(x=None), dict(packed=None), dict(out=None), dict(offsets=None), dict(x_rows=0), dict(places=0), dict(experts=0),
        dict(cols=0), dict(k=0), dict(top_k=0), dict(x_dtype=F32), dict(x_stride=32), dict(order=0, x_rows=39),
        dict(out_dtype=9), dict(out_stride=63), dict(out=P + 1), dict(swiglu=0, out_dtype=MX4), dict(packed_bytes=100),
        dict(out_dtype=MX4, out=P + 8), dict(out_dtype=MX4, out_bytes=100), dict(workspace=None), dict(workspace_bytes=9)]),
    ("hi_rocm_mx4_grouped_product", UNSUPPORTED, [
        dict(cols=96), dict(k=48), dict(experts=2049), dict(places=(1 << 22) + 1), dict(x=P + 4), dict(x_stride=72 + 4),
        dict(x_rows=1 << 23)]),
]


@pytest.mark.parametrize("name,status,changed", [(n, s, c) for n, s, cs in REFUSED for c in cs],
                         ids=lambda v: "-".join(v) if isinstance(v, dict) else str(v))
def test_refused(name, status, changed):
    args = dict(GOOD[name])
    for key, v in changed.items():
        assert key in args, key
        args[key] = v
    assert getattr(_lib.load(), name)(*args.values()) == status
    assert _lib.load().hi_rocm_last_error().decode().startswith(name + ":")


def _bytes(name, *args, status=0):
    out = ctypes.c_size_t()
    assert getattr(_lib.load(), name)(*args, ctypes.byref(out)) == status
    return out.value


def test_sizes():
    lib = _lib.load()
    name = "hi_rocm_spec_sampled_workspace_bytes"
    sizes = [_bytes(name, b, v) for b, v in ((1, 1), (1, 50257), (1, 151936), (64, 151936), (65535, 151936))]
    assert sizes == sorted(sizes) and sizes[0] > 0
    for bad in ((0, 10), (-1, 10), (1, 0)):
        _bytes(name, *bad, status=ARGS)
    for bad in ((65536, 10), (1, (1 << 23) + 1)):
        _bytes(name, *bad, status=UNSUPPORTED)
    # rows: codes, then the scales of whole quads
    for rows, k in ((1, 32), (3, 1184), (8192, 4096)):
        assert _bytes("hi_rocm_mx4_rows_bytes", rows, k) >= rows * (k // 2 + 16 * -(-k // 512))
    for e, n, k in ((1, 1, 32), (1, 151936, 4096), (60, 1000, 1184)):
        tiles, steps, quads = -(-n // 16), -(-k // 128), -(-k // 512)
        assert _bytes("hi_rocm_mx4_packed_bytes", e, n, k) >= e * tiles * (1024 * steps + 256 * quads)
    # few rows need no workspace
    name = "hi_rocm_mx4_workspace_bytes"
    assert _bytes(name, 1, 1, 65536) == 0 and _bytes(name, 16, 16, 4096) == 0 and _bytes(name, 8, 64, 2048) == 0
    assert _bytes(name, 17, 17, 64) == _bytes("hi_rocm_mx4_rows_bytes", 17, 64)
    assert _bytes(name, 16, 16, 8192) == _bytes("hi_rocm_mx4_rows_bytes", 16, 8192)
    assert _bytes(name, 2, 64, 65536) == _bytes("hi_rocm_mx4_rows_bytes", 2, 65536)
    # a linear layer of few columns rounds more rows on the way, of no more than 4,096 inputs
    name = "hi_rocm_mx4_linear_workspace_bytes"
    assert _bytes(name, 1, 151936, 65536) == 0 and _bytes(name, 16, 48, 4096) == 0 and _bytes(name, 64, 1000, 1184) == 0
    for rows, n, k in ((500, 16384, 512), (17, 48, 4128), (64, 32000, 1024), (16, 48, 8192)):
        assert _bytes(name, rows, n, k) == _bytes("hi_rocm_mx4_rows_bytes", rows, k)
    for name, good in (("hi_rocm_mx4_rows_bytes", (4, 64)), ("hi_rocm_mx4_packed_bytes", (1, 4, 64)),
                       ("hi_rocm_mx4_linear_workspace_bytes", (4, 4, 64)),
                       ("hi_rocm_mx4_workspace_bytes", (4, 4, 64))):
        assert getattr(lib, name)(*good, None) == ARGS
        _bytes(name, *good[:-1], 48, status=UNSUPPORTED)
        _bytes(name, *good[:-1], 0, status=ARGS)
        _bytes(name, 0, *good[1:], status=ARGS)


def test_fronts_need_a_gpu():
    """Calls whose tensors are on the CPU go no further than the front end."""
    x, codes, scales = torch.zeros(4, 64), torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    verifier = SpecVerifier(2, 1, 10, device="cpu")
    out = verifier.outputs(2)
    t, u = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 2)
    calls = [lambda: mx4.quantize_mx4(x), lambda: mx4.quantize_mx4(x, out=(codes, scales)),
             lambda: mx4.dequantize_mx4(codes, scales), lambda: mx4.mx4_rows(x), lambda: mx4.Mx4Linear(codes, scales),
             lambda: mx4.Mx4Experts(codes.view(1, 4, 32), scales.view(1, 4, 2), codes[:, :16].contiguous().view(1, 4, 16),
                                    scales[:, :1].contiguous().view(1, 4, 1), 4, 1),
             lambda: verifier(torch.zeros(2, 2, 10), t, u, out=out),
             lambda: verifier(torch.zeros(2, 2, 10), t, u, draft_probs=torch.zeros(2, 1, 10), out=out)]
    for call in calls:
        with pytest.raises(ValueError):
            call()


def test_rounding_oracle():
    """The oracle's rounding, by hand: a block's scale from its largest value, ties
    to even codes, saturation, zeros, subnormal blocks, blocks that are not finite."""
    x = torch.zeros(7, 32)
    x[0, :8] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, -5.0])  # scale 1
    x[1, :3] = torch.tensor([7.9, 6.0, -7.9])                               # 8 is the next scale's
    x[2, :3] = torch.tensor([8.0, 1.0, 0.5])                                # scale 2
    x[4, 0] = float("inf")
    x[5, 0] = 2.0 ** -140
    x[6, 0] = 3.0e38
    codes, scales = mx4_oracle.quantize(x)
    assert codes[0, :8].tolist() == [6, 0, 2, 2, 4, 4, 6, 14]
    assert codes[1, :3].tolist() == [7, 7, 15]
    assert codes[2, :3].tolist() == [6, 1, 0]
    assert scales[:, 0].tolist() == [127, 127, 128, 0, 255, 0, 252]
    v = mx4_oracle.values(mx4_oracle.pack_nibbles(codes), scales)
    assert v[0, :8].tolist() == [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, -4.0] and v[2, 1] == 1.0 and v[4].isnan().all()
    assert (v[3] == 0).all() and v[5, 0] == 0 and v[6, 0] == 6 * 2.0 ** 125


def test_verification_oracle():
    """The oracle's rule, by hand."""
    import numpy as np
    p = np.array([[[0.5, 0.5, 0.0], [0.2, 0.2, 0.6]]])
    q = np.array([[[0.25, 0.75, 0.0]]])

    def run(t, u0, u1, draft=q, lengths=None):
        out, n = spec_sampled_oracle.verify(p, np.array([[t]]), np.array([[u0, u1]]), draft, lengths)
        return out[0].tolist(), int(n[0])

    assert run(0, 0.99, 0.3) == ([0, 1], 2)      # p / q = 2: always accepted; 0.2 <= 0.3 < 0.4
    assert run(1, 0.66, 0.5) == ([1, 2], 2)      # 0.66 * 0.75 < 0.5
    assert run(1, 0.67, 0.99) == ([0, -1], 1)    # rejected: only token 0 has more of p
    assert run(2, 0.0, 0.0) == ([0, -1], 1)      # no probability: rejected
    assert run(1, 0.4, 0.0, draft=None) == ([1, 0], 2)
    assert run(1, 0.5, 0.9, draft=None) == ([0, -1], 1)
    assert run(7, 0.0, 0.9) == ([0, -1], 1)      # no token
    assert run(0, 0.0, 0.7, lengths=[0]) == ([1, -1], 1)
