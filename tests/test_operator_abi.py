"""CPU checks of the C ABI of the beam, 4-bit and expert entry points: sizes
of workspaces and packed weights, and bad arguments refused before any HIP
call."""
import ctypes

import pytest

from hi_amd import _lib

ARGS, UNSUPPORTED = _lib.ERR_ARGS, _lib.ERR_UNSUPPORTED
F32, BF16 = _lib.DTYPE_F32, _lib.DTYPE_BF16
P = 1 << 32  # an address on 16 bytes that nothing may touch


def _call(name, **changed):
    """The entry point with arguments that pass its checks, but for `changed`."""
    args = dict(GOOD[name])
    for k, v in changed.items():
        assert k in args, k
        args[k] = v
    rc = getattr(_lib.load(), name)(*args.values())
    return rc, _lib.load().hi_rocm_last_error().decode()


GOOD = {
    "hi_rocm_beam_select": dict(
        logits=P, dtype=F32, batch=2, beams=4, vocab=1000, row_stride=1000, scores=P, finished=0, eos=2, mask=0,
        n_out=4, out_scores=P, out_tokens=P, out_parents=P, out_finished=P, workspace=P, workspace_bytes=1 << 30,
        stream=None),
    "hi_rocm_beam_reorder": dict(
        src=P, dst=P, parents=P, batch=2, beams=4, outer=3, outer_stride=8 * 2 * 4096, row_stride=2 * 4096, mid=2,
        mid_stride=4096, positions=16, pos_bytes=256, lengths=0, stream=None),
    "hi_rocm_w4_pack": dict(q=P, scales=P, zeros=0, scale_dtype=BF16, n=64, k=256, group=64, packed=P,
                            packed_bytes=1 << 30, stream=None),
    "hi_rocm_w4_linear": dict(
        x=P, rows=2, x_stride=256, packed=P, packed_bytes=1 << 30, scale_dtype=BF16, has_zeros=0, n=64, k=256,
        group=64, bias=0, out=P, out_dtype=F32, out_stride=64, stream=None),
    "hi_rocm_moe_group": dict(ids=P, tokens=4, top_k=2, experts=8, order=P, slots=P, offsets=P, stream=None),
    "hi_rocm_moe_grouped_product": dict(
        x=P, x_rows=4, x_stride=64, order=P, top_k=2, offsets=P, places=8, experts=8, weight=P, cols=32, k=64,
        swiglu=0, out=P, out_dtype=BF16, out_stride=32, stream=None),
    "hi_rocm_moe_combine": dict(
        y=P, y_dtype=F32, y_stride=32, slots=P, offsets=P, experts=8, weights=P, tokens=4, top_k=2, cols=32, out=P,
        out_dtype=BF16, out_stride=32, stream=None),
}

REFUSED = [
    ("hi_rocm_beam_select", ARGS, [
        dict(logits=None), dict(scores=None), dict(out_scores=None), dict(out_tokens=None), dict(out_parents=None),
        dict(out_finished=None), dict(workspace=None), dict(workspace=P + 8), dict(workspace_bytes=16), dict(batch=0),
        dict(beams=0), dict(vocab=0), dict(n_out=0), dict(batch=-1), dict(row_stride=999), dict(dtype=7),
        dict(logits=P + 2), dict(logits=P + 1, dtype=BF16), dict(finished=P, eos=_lib.BEAM_NO_EOS)]),
    ("hi_rocm_beam_select", UNSUPPORTED, [
        dict(beams=33), dict(n_out=65), dict(batch=16384), dict(vocab=(1 << 23) + 1, row_stride=1 << 24)]),
    ("hi_rocm_beam_reorder", ARGS, [
        dict(src=None), dict(dst=None), dict(parents=None), dict(batch=0), dict(beams=0), dict(outer=0), dict(mid=0),
        dict(positions=0), dict(pos_bytes=0), dict(row_stride=-1), dict(mid_stride=4095), dict(row_stride=4096),
        dict(outer_stride=8 * 2 * 4096 - 1), dict(dst=P + 256), dict(dst=P - 3 * 8 * 2 * 4096 + 16)]),
    ("hi_rocm_beam_reorder", UNSUPPORTED, [
        dict(beams=33, outer_stride=1 << 40), dict(batch=65536, outer_stride=1 << 44), dict(positions=1 << 50),
        dict(outer=1 << 47), dict(outer_stride=1 << 47), dict(outer=1 << 23, outer_stride=1 << 20, mid=2),
        # 2^24 pieces of 256 units a row: by bytes, by 16 bytes
        dict(pos_bytes=1, positions=1 << 32, outer=1, mid=1, batch=1, beams=1, row_stride=1 << 33, mid_stride=1 << 33),
        dict(pos_bytes=16, positions=1 << 32, outer=1, mid=1, batch=1, beams=1)]),
    ("hi_rocm_w4_pack", ARGS, [
        dict(q=None), dict(scales=None), dict(packed=None), dict(packed=P + 8), dict(packed_bytes=64), dict(n=0),
        dict(k=0), dict(group=0), dict(scale_dtype=9), dict(scales=P + 1), dict(zeros=P + 1),
        dict(scales=P + 2, scale_dtype=F32)]),
    ("hi_rocm_w4_pack", UNSUPPORTED, [
        dict(group=16), dict(group=96, k=288), dict(k=250), dict(n=(1 << 24) + 1), dict(k=1 << 25),
        dict(n=1 << 18, k=1 << 18, packed_bytes=1 << 50)]),
    ("hi_rocm_w4_linear", ARGS, [
        dict(x=None), dict(packed=None), dict(out=None), dict(rows=0), dict(x_stride=255), dict(out_stride=63),
        dict(out_dtype=5), dict(scale_dtype=5), dict(packed=P + 8), dict(packed_bytes=4096), dict(out=P + 2),
        dict(out=P + 1, out_dtype=BF16), dict(bias=P + 2)]),
    ("hi_rocm_w4_linear", UNSUPPORTED, [
        dict(group=48, k=288, x_stride=288), dict(k=192, group=128), dict(rows=16 * 65535 + 1), dict(x=P + 8),
        dict(x_stride=260)]),
    ("hi_rocm_moe_group", ARGS, [
        dict(ids=None), dict(order=None), dict(slots=None), dict(offsets=None), dict(tokens=0), dict(top_k=0),
        dict(experts=0)]),
    ("hi_rocm_moe_group", UNSUPPORTED, [dict(experts=2049), dict(tokens=(1 << 21) + 1)]),
    ("hi_rocm_moe_grouped_product", ARGS, [
        dict(x=None), dict(offsets=None), dict(weight=None), dict(out=None), dict(x_rows=0), dict(places=0),
        dict(experts=0), dict(cols=0), dict(k=0), dict(x_stride=56), dict(out_dtype=4), dict(top_k=0),
        dict(order=0, x_rows=7), dict(swiglu=1, cols=33), dict(out_stride=31), dict(swiglu=1, out_stride=15),
        dict(out=P + 1), dict(out=P + 2, out_dtype=F32)]),
    ("hi_rocm_moe_grouped_product", UNSUPPORTED, [
        dict(experts=2049), dict(places=(1 << 22) + 1), dict(cols=(1 << 20) + 1, out_stride=1 << 21),
        dict(k=60), dict(x_stride=68), dict(x=P + 8), dict(weight=P + 8),
        dict(places=1 << 22, cols=1 << 20, out_stride=1 << 20, experts=2048)]),
    ("hi_rocm_moe_combine", ARGS, [
        dict(y=None), dict(slots=None), dict(offsets=None), dict(weights=None), dict(out=None), dict(tokens=0),
        dict(top_k=0), dict(experts=0), dict(cols=0), dict(y_stride=31), dict(out_stride=31), dict(y_dtype=4),
        dict(out_dtype=4), dict(y=P + 2), dict(out=P + 1)]),
    ("hi_rocm_moe_combine", UNSUPPORTED, [
        dict(experts=2049), dict(tokens=(1 << 21) + 1), dict(cols=(1 << 20) + 1, y_stride=1 << 21, out_stride=1 << 21)]),
]


@pytest.mark.parametrize("name,status,changed", [(n, s, c) for n, s, cs in REFUSED for c in cs],
                         ids=lambda v: "-".join(v) if isinstance(v, dict) else str(v))
def test_refused(name, status, changed):
    rc, message = _call(name, **changed)
    assert rc == status
    assert message.startswith(name + ":")


def test_beam_workspace_bytes():
    lib, out = _lib.load(), ctypes.c_size_t()

    def bytes_of(*a):
        assert lib.hi_rocm_beam_workspace_bytes(*a, ctypes.byref(out)) == 0
        return out.value

    assert 0 < bytes_of(1, 1, 1, 1) <= bytes_of(1, 4, 151936, 8) < bytes_of(64, 8, 151936, 8) < bytes_of(64, 8, 151936, 16)
    # enough for any smaller batch too
    sizes = [bytes_of(b, 8, 50257, 16) for b in (1, 2, 16, 40, 63, 64, 65, 100, 200)]
    assert sizes == sorted(sizes)
    assert bytes_of(65535, 1, 8, 1) > 0
    for a in ((0, 4, 10, 4), (1, 0, 10, 4), (1, 4, 0, 4), (1, 4, 10, 0)):
        assert lib.hi_rocm_beam_workspace_bytes(*a, ctypes.byref(out)) == ARGS
    assert lib.hi_rocm_beam_workspace_bytes(1, 4, 10, 4, None) == ARGS
    for a in ((1, 33, 10, 4), (1, 4, 10, 65), (65536, 1, 10, 1), (1, 4, (1 << 23) + 1, 4)):
        assert lib.hi_rocm_beam_workspace_bytes(*a, ctypes.byref(out)) == UNSUPPORTED


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype,size", [(F32, 4), (BF16, 2)])
@pytest.mark.parametrize("zeros", [0, 1])
def test_packed_bytes(group, dtype, size, zeros):
    lib, out = _lib.load(), ctypes.c_size_t()
    for n, k in ((1, group), (16, 128), (1000, 37 * group), (151936, 4096)):
        assert lib.hi_rocm_w4_packed_bytes(n, k, group, dtype, zeros, ctypes.byref(out)) == 0
        blocks = -(-n // 16) * -(-k // 128)
        need = blocks * (1024 + (1 + zeros) * 16 * (128 // group) * size)
        assert need <= out.value < need + 3 * 256
    assert lib.hi_rocm_w4_packed_bytes(16, group + 8, group, dtype, zeros, ctypes.byref(out)) == UNSUPPORTED
    assert lib.hi_rocm_w4_packed_bytes(0, group, group, dtype, zeros, ctypes.byref(out)) == ARGS
    assert lib.hi_rocm_w4_packed_bytes(16, group, group, dtype, zeros, None) == ARGS
