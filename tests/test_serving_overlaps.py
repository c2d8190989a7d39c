"""What the serving step's calls write overlaps nothing else of the call: refused before any device
work.  Memory that only lies between another's rows is none of it, and no call is refused for it."""
import ctypes

import pytest

from sile_amd import _abi
from tests.test_serving_abi import APPEND, CHUNK, LOGPROBS, NORM, P, ROPE, refused


def passes(f, **kw):
    """The checks let the call pass, which without a GPU ends at its first look at the device."""
    count = ctypes.c_int(0)
    _abi.call("sile_hip_device_count", ctypes.byref(count))
    if count.value:
        pytest.skip("made-up addresses: only where no kernel can run")
    with pytest.raises(_abi.SileError) as e:
        f(**kw)
    assert e.value.kind != "Shape", str(e.value)


# tokens of a fused projection: 4 query heads, 2 key heads and 2 value heads of 64, 512 elements of 2 bytes
FUSED = dict(q=P, ldq=512, k=P + 512, ldk=512)


def test_rope():
    f = _abi.rope
    for change in (dict(q_out=3 * P), dict(q_out=3 * P + 64), dict(k_out=P), dict(k_out=P + 3 * 512 + 256), dict(k_out=2 * P),
                   dict(q_out=4 * P - 512), dict(q_out=5 * P - 1536), dict(k_out=5 * P), dict(q_out=6 * P), dict(k_out=6 * P - 1008),
                   {**FUSED, "k_out": P + 256, "ldko": 512}, {**FUSED, "q_out": P + 256, "ldqo": 512},
                   {**FUSED, "q_out": P, "ldqo": 512, "k_out": P + 384, "ldko": 512},
                   {**FUSED, "q_out": P + 640, "ldqo": 1024}):
        refused("Shape", f, **{**ROPE, **change})


def test_rope_between_rows():
    f = _abi.rope
    for change in ({**FUSED, "q_out": P, "ldqo": 512, "k_out": P + 512, "ldko": 512},   # in place
                   {**FUSED, "k_out": P + 768, "ldko": 512},                            # over the values
                   {**FUSED, "k_out": P + 768, "ldko": 1024},                           # over every other token's
                   dict(q=P, ldq=512, q_out=P + 512, ldqo=512),
                   dict(q_out=3 * P - 2048), dict(q_out=3 * P + 1024)):                 # end to end
        passes(f, **{**ROPE, **change})


def test_rope_append():
    f = _abi.rope_append
    page = 2048 * 2
    for change in (dict(q_out=3 * P), dict(q_out=4 * P + 256), dict(q_out=5 * P), dict(q_out=6 * P), dict(q_out=7 * P + 512),
                   dict(q_out=8 * P + 9 * page), dict(q_out=9 * P), dict(rows=2 * P), dict(v_pages=7 * P), dict(v_pages=7 * P + 9 * page),
                   dict(k_pages=P), dict(v_pages=P + 512), dict(k_pages=3 * P), dict(v_pages=4 * P), dict(k_pages=5 * P), dict(v_pages=6 * P),
                   dict(k_pages=9 * P), dict(k_pages=4 * P - 9 * page), dict(rows=8 * P),
                   dict(page_stride=2 * 2048, v_pages=7 * P + page // 2), dict(page_stride=3 * 2048, v_pages=7 * P + 2 * page + 16)):
        refused("Shape", f, **{**APPEND, **change})


def test_rope_append_between_rows():
    f = _abi.rope_append
    page = 2048 * 2
    for change in (dict(page_stride=2 * 2048, v_pages=7 * P + page),                   # K and V of a page side by side
                   dict(page_stride=2 * 2048, k_pages=7 * P + page, v_pages=7 * P),
                   dict(q=P, ldq=512, k=P + 512, ldk=512, v=P + 768, ldv=512),         # a fused projection
                   dict(q=P, ldq=512, q_out=P, ldqo=512, k=P + 512, ldk=512, v=P + 768, ldv=512),
                   dict(num_pages=0, v_pages=7 * P), dict(q_heads=0, q_out=3 * P), dict(v_pages=7 * P + 10 * page)):
        passes(f, **{**APPEND, **change})


def test_rows_as_sets():
    """Whether rows of any pitch share a byte, against counting them."""
    import random
    rng = random.Random(3)
    seen = [0, 0]
    for _ in range(3000):
        n, width = rng.randint(1, 6), 2 * rng.randint(1, 4)
        lx, ly = width + rng.randint(0, 20), width + rng.randint(0, 20)
        off = rng.randint(-60, 60)
        if off == 0 and lx == ly:
            continue
        rows = lambda at, ld: {at + i * ld + j for i in range(n) for j in range(width)}   # noqa: E731
        want = bool(rows(0, lx) & rows(off, ly))
        seen[want] += 1
        kw = dict(dtype=_abi.F32, layout=0, n_tokens=n, q_heads=1, kv_heads=0, head_dim=width, rot_dim=width, q=P, ldq=lx,
                  q_out=P + 4 * off, ldqo=ly, k=0, ldk=0, k_out=0, ldko=0, positions=5 * P, turns=6 * P)
        if want:
            refused("Shape", _abi.rope, **kw)
        else:
            passes(_abi.rope, **kw)
    assert min(seen) > 500


def test_chunk():
    f = _abi.paged_attn_chunk
    page = 2048 * 2
    for change in (dict(o=P), dict(o=P + 29 * 512), dict(o=2 * P), dict(o=3 * P + page), dict(o=4 * P + 9 * page), dict(o=5 * P - 512),
                   dict(o=6 * P), dict(o=3 * P - 29 * 512), dict(q=P, ldq=512, o=P + 256, ldo=1024),
                   dict(page_stride=2 * 2048, o=3 * P + page, ldo=256)):
        refused("Shape", f, **{**CHUNK, **change})
    for change in (dict(q=P, ldq=512, o=P + 512, ldo=512), dict(o=P + 30 * 512), dict(o=4 * P - 30 * 512), dict(o=4 * P + 10 * page),
                   dict(page_stride=2 * 2048, v_pages=3 * P + page), dict(num_pages=0, o=3 * P)):
        passes(f, **{**CHUNK, **change})


@pytest.mark.gpu
def test_chunk_workspace(hip):
    """A workspace over any operand of the call (its size is the device's to say).  Operands and workspaces
    all lie in one allocation."""
    need = hip.paged_attn_chunk_workspace(4, 30, 4, 2, 64)
    far = (need + (1 << 20)) // 16 * 16
    arena = hip.DeviceBuffer(10 * far)
    arena.fill_bytes(0)
    x = lambda i: arena.ptr + i * far   # noqa: E731
    base = dict(q=x(1), starts=x(2), k_pages=x(3), v_pages=x(4), tables=x(5), lengths=x(6), o=x(7), workspace_bytes=need)
    for at, over in ((1, 16), (2, 0), (3, 4096), (4, 9 * 4096), (5, 32), (6, 0), (7, 256)):
        refused("Shape", hip.paged_attn_chunk, **{**CHUNK, **base, "workspace": x(at) + over})
        refused("Shape", hip.paged_attn_chunk, **{**CHUNK, **base, "workspace": x(at) - need + 16})
    arena.close()


DECODE = {k: v for k, v in CHUNK.items() if k not in ("n_rows", "n_tokens", "starts")}


def test_decode():
    f = _abi.paged_attn_decode
    page = 2048 * 2
    base = {**DECODE, "batch": 4}
    for change in (dict(o=P), dict(o=P + 3 * 512), dict(o=3 * P + page), dict(o=4 * P + 9 * page), dict(o=5 * P - 512), dict(o=6 * P),
                   dict(q=P, ldq=512, o=P + 256, ldo=1024)):
        refused("Shape", f, **{**base, **change})
    for change in (dict(q=P, ldq=512, o=P + 512, ldo=512), dict(o=P + 4 * 512), dict(o=4 * P - 4 * 512), dict(num_pages=0, o=3 * P)):
        passes(f, **{**base, **change})


@pytest.mark.gpu
def test_decode_workspace(hip):
    need = hip.paged_attn_workspace(4, 4, 2, 64)
    far = (need + (1 << 20)) // 16 * 16
    arena = hip.DeviceBuffer(10 * far)
    arena.fill_bytes(0)
    x = lambda i: arena.ptr + i * far   # noqa: E731
    base = {**DECODE, "batch": 4, "q": x(1), "k_pages": x(3), "v_pages": x(4), "tables": x(5), "lengths": x(6), "o": x(7),
            "workspace_bytes": need}
    for at, over in ((1, 16), (3, 4096), (4, 9 * 4096), (5, 32), (6, 0), (7, 256)):
        refused("Shape", hip.paged_attn_decode, **{**base, "workspace": x(at) + over})
        refused("Shape", hip.paged_attn_decode, **{**base, "workspace": x(at) - (need + 15) // 16 * 16 + 16})
    arena.close()


def test_norm_between_rows():
    """Rows of 64 elements of 2 bytes, in slices of wider ones."""
    f = _abi.rmsnorm_rows
    wide = dict(x=P, ldx=256, residual=P + 128, ldr=256)
    for change in ({**wide, "sum_out": P + 256, "lds": 256, "y": P + 384, "ldy": 256}, {**wide, "sum_out": P + 128, "lds": 256, "y": P, "ldy": 256},
                   {**wide, "y": P, "ldy": 256}, {**wide, "out_type": _abi.F8E4M3, "y": P + 256, "ldy": 512},
                   {**wide, "out_type": _abi.F8E4M3, "y": P + 448, "ldy": 1024, "group": 16, "scales": 6 * P}):
        passes(f, **{**NORM, **change})
    for change in ({**wide, "y": P + 64, "ldy": 256}, {**wide, "sum_out": P + 256, "lds": 256, "y": P + 320, "ldy": 256},
                   {**wide, "out_type": _abi.F8E4M3, "y": P, "ldy": 512}, {**wide, "out_type": _abi.F8E4M3, "y": P + 450, "ldy": 300},
                   {**wide, "sum_out": P, "lds": 128}, {**wide, "weight": P, "y": P, "ldy": 256}):
        refused("Shape", f, **{**NORM, **change})


def test_logprobs_between_rows():
    """Outputs behind the columns of padded rows."""
    f = _abi.logprobs_rows
    for change in (dict(ldx=164, logp=P + 400, entropy=P + 416, top_logp=P + 432), dict(top_k=0, top_logp=P, top_ids=P), dict(logp=None, targets=3 * P, entropy=4 * P)):
        passes(f, **{**LOGPROBS, **change})
    for change in (dict(ldx=164, logp=P + 644), dict(ldx=164, top_ids=P + 656 + 400 - 76)):
        refused("Shape", f, **{**LOGPROBS, **change})


@pytest.mark.gpu
def test_norm_of_slices(hip):
    """Sum and result of a slice of wide rows to other slices of them, as to arrays of their own."""
    import numpy as np
    x = np.random.default_rng(0).normal(size=(50, 4, 256)).astype(np.float32)
    wide, apart = hip.DeviceBuffer.from_array(x), hip.DeviceBuffer(50 * 512 * 4)
    args = (hip.F32, hip.F32, 50, 256, wide.ptr, 1024, wide.ptr + 1024, 1024)
    hip.rmsnorm_rows(*args, apart.ptr, 512, 0, 1e-5, apart.ptr + 1024, 512)
    hip.rmsnorm_rows(*args, wide.ptr + 2 * 1024, 1024, 0, 1e-5, wide.ptr + 3 * 1024, 1024)
    hip.synchronize()
    got, want = wide.download(np.float32, (50, 4, 256)), apart.download(np.float32, (50, 2, 256))
    assert np.array_equal(got[:, 2:], want) and np.array_equal(got[:, :2], x[:, :2])
