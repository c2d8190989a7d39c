"""The serving step's entry points without a GPU: refusals come before any device work, and the
turns of rotary positions are what their formulas say."""
import numpy as np
import pytest

from sile_amd import _abi
from tests import serving_ref as ref

P = 1 << 20   # an address that no refused call looks at


def refused(kind, call, *args, **kw):
    with pytest.raises(_abi.SileError) as e:
        call(*args, **kw)
    assert e.value.kind == kind, str(e.value)


@pytest.mark.parametrize("rot", [0, 2, 4, 32, 128, 2048])
def test_turns(rot):
    a = _abi
    for base in (10000.0, 500000.0):
        for code, name, args in ((a.ROPE_UNSCALED, "none", ()), (a.ROPE_LINEAR, "linear", (4.0,)), (a.ROPE_BASE, "base", (8.0,)),
                                 (a.ROPE_TURNS, "turns", (8.0, 8192.0, 1.0, 4.0)), (a.ROPE_DIMS, "dims", (16.0, 4096.0, 1.0, 32.0))):
            got, want = a.rope_turns(code, rot, base, *args), ref.turns(name, rot, base, *args)
            assert np.allclose(got, want, rtol=1e-12, atol=0), name


def test_turns_ends():
    """The fastest pair keeps its turns, the slowest has 1 / factor of them."""
    a = _abi
    plain = a.rope_turns(a.ROPE_UNSCALED, 128, 1e4)
    assert plain[0] == 1 / (2 * np.pi)
    for code, args in ((a.ROPE_BASE, ()), (a.ROPE_TURNS, (4096.0, 1.0, 32.0)), (a.ROPE_DIMS, (4096.0, 1.0, 32.0))):
        t = a.rope_turns(code, 128, 1e4, 4.0, *args)
        assert np.isclose(t[0], plain[0]) and np.isclose(t[-1], plain[-1] / 4)
        assert (np.diff(t) < 0).all()


def test_turns_refused():
    a = _abi
    refused("Shape", a.rope_turns, a.ROPE_UNSCALED, 3, 1e4)
    refused("Shape", a.rope_turns, a.ROPE_UNSCALED, 4096, 1e4)
    refused("Shape", a.rope_turns, a.ROPE_UNSCALED, 64, 0.0)
    refused("Shape", a.rope_turns, a.ROPE_UNSCALED, 64, float("nan"))
    refused("Shape", a.rope_turns, a.ROPE_LINEAR, 64, 1e4, 0.0)
    refused("Shape", a.rope_turns, a.ROPE_TURNS, 64, 1e4, 4.0, 0.0, 1.0, 4.0)
    refused("Shape", a.rope_turns, a.ROPE_TURNS, 64, 1e4, 4.0, 4096.0, 4.0, 4.0)
    refused("Shape", a.rope_turns, a.ROPE_DIMS, 64, 1.0, 4.0, 4096.0, 1.0, 4.0)
    refused("Shape", a.rope_turns, 5, 64, 1e4)


def test_slots_refused():
    f = _abi.kv_slots
    ok = dict(n_rows=4, lengths=P, need=2 * P, granted=0, max_tokens=8, starts=3 * P, rows=4 * P, positions=5 * P, lengths_out=6 * P)
    for change in (dict(n_rows=-1), dict(n_rows=65537), dict(max_tokens=-1), dict(max_tokens=2 ** 31), dict(lengths=None), dict(need=None),
                   dict(starts=None), dict(rows=None), dict(positions=None), dict(lengths_out=None), dict(lengths_out=P),
                   dict(lengths_out=P + 12), dict(rows=5 * P + 16), dict(starts=P), dict(granted=4 * P), dict(positions=2 * P)):
        refused("Shape", f, **{**ok, **change})


ROPE = dict(dtype=_abi.BF16, layout=0, n_tokens=4, q_heads=4, kv_heads=2, head_dim=64, rot_dim=64, q=P, ldq=256, q_out=2 * P, ldqo=256,
            k=3 * P, ldk=128, k_out=4 * P, ldko=128, positions=5 * P, turns=6 * P, magnitude=1.0)


def test_rope_refused():
    f = _abi.rope
    refused("UnsupportedBackend", f, **{**ROPE, "dtype": _abi.F8E4M3})
    refused("UnsupportedBackend", f, **{**ROPE, "head_dim": 4096, "ldq": 1 << 20, "ldqo": 1 << 20, "ldk": 1 << 20, "ldko": 1 << 20})
    for change in (dict(layout=2), dict(n_tokens=-1), dict(q_heads=-1), dict(q_heads=0, kv_heads=0), dict(rot_dim=63), dict(rot_dim=66),
                   dict(rot_dim=-2), dict(q=None), dict(q_out=None), dict(k=None), dict(k_out=None), dict(positions=None), dict(turns=None),
                   dict(ldq=255), dict(ldqo=255), dict(ldk=127), dict(ldko=127), dict(q=P + 1), dict(k_out=P + 1), dict(q_out=P + 64),
                   dict(q_out=P, ldqo=264), dict(k_out=3 * P + 512), dict(magnitude=float("nan")), dict(magnitude=float("inf")),
                   dict(ldq=1 << 50)):
        refused("Shape", f, **{**ROPE, **change})


APPEND = dict(dtype=_abi.BF16, cache_type=_abi.BF16, layout=0, n_tokens=4, q_heads=4, kv_heads=2, head_dim=64, rot_dim=64, q=P, ldq=256,
              q_out=2 * P, ldqo=256, k=3 * P, ldk=128, v=4 * P, ldv=128, rows=0, positions=5 * P, turns=6 * P, magnitude=1.0,
              k_pages=7 * P, v_pages=8 * P, num_pages=10, page_size=16, page_stride=2048, tables=9 * P, n_rows=4, ld_table=2)


def test_rope_append_refused():
    f = _abi.rope_append
    for change in (dict(dtype=_abi.F32), dict(cache_type=_abi.F16), dict(head_dim=72, cache_type=_abi.F8E4M3), dict(head_dim=264)):
        refused("UnsupportedBackend", f, **{**APPEND, **change})
    for change in (dict(layout=-1), dict(n_tokens=-1), dict(rot_dim=66), dict(q=None), dict(k=None), dict(v=None), dict(positions=None),
                   dict(turns=None), dict(k_pages=None), dict(v_pages=None), dict(tables=None), dict(ldk=127), dict(ldv=120), dict(ldk=132),
                   dict(q=P + 2), dict(k=3 * P + 8), dict(k_pages=7 * P + 8), dict(page_size=24), dict(page_stride=2047), dict(kv_heads=0),
                   dict(num_pages=-1), dict(n_rows=-1), dict(ld_table=-1), dict(q_out=P + 16), dict(magnitude=float("nan"))):
        refused("Shape", f, **{**APPEND, **change})


NORM = dict(in_type=_abi.BF16, out_type=_abi.BF16, rows=4, cols=64, x=P, ldx=64, residual=2 * P, ldr=64, sum_out=3 * P, lds=64,
            weight=4 * P, eps=1e-5, y=5 * P, ldy=64, scale=1.0, scales=0, group=0)


def test_norm_refused():
    f = _abi.rmsnorm_rows
    refused("UnsupportedBackend", f, **{**NORM, "in_type": _abi.F8E4M3})
    refused("UnsupportedBackend", f, **{**NORM, "out_type": _abi.F32})
    for change in (dict(rows=-1), dict(cols=-1), dict(cols=1 << 31), dict(x=None), dict(y=None), dict(ldx=63), dict(ldr=63), dict(lds=63),
                   dict(ldy=63), dict(group=64), dict(group=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(x=P + 1), dict(y=5 * P + 1),
                   dict(weight=4 * P + 1), dict(y=3 * P), dict(y=P + 2), dict(sum_out=P + 128), dict(sum_out=2 * P, lds=72),
                   dict(y=P, ldy=72), dict(sum_out=4 * P), dict(y=4 * P), dict(ldx=1 << 50),
                   dict(out_type=_abi.F8E4M3, group=48), dict(out_type=_abi.F8E4M3, group=16), dict(out_type=_abi.F8E4M3, y=P),
                   dict(out_type=_abi.F8E4M3, group=16, scales=5 * P), dict(out_type=_abi.F8E4M3, group=16, scales=6 * P + 2),
                   dict(out_type=_abi.F8E4M3, group=16, scales=P), dict(out_type=_abi.F8E4M3, group=16, scales=3 * P)):
        refused("Shape", f, **{**NORM, **change})


LOGPROBS = dict(in_type=_abi.F32, rows=4, cols=100, x=P, ldx=100, scale=1.0, targets=2 * P, logp=3 * P, entropy=4 * P, top_k=5,
                top_logp=5 * P, top_ids=6 * P)


def test_logprobs_refused():
    f = _abi.logprobs_rows
    refused("UnsupportedBackend", f, **{**LOGPROBS, "in_type": _abi.F8E4M3})
    for change in (dict(rows=-1), dict(rows=1 << 23), dict(cols=-1), dict(cols=1 << 31), dict(top_k=-1), dict(top_k=65), dict(scale=0.0),
                   dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(x=None), dict(targets=None), dict(top_logp=None),
                   dict(top_ids=None), dict(ldx=99), dict(ldx=1 << 60), dict(x=P + 2), dict(logp=3 * P + 2), dict(logp=P + 16),
                   dict(entropy=3 * P + 8), dict(top_ids=5 * P + 64), dict(logp=2 * P)):
        refused("Shape", f, **{**LOGPROBS, **change})
    refused("Shape", _abi.logprobs_workspace, 4, 100, 65)
    refused("Shape", _abi.logprobs_workspace, -1, 100, 5)
    assert _abi.status("sile_hip_logprobs_workspace", 4, 100, 5, None) == 5


def test_nothing_to_do():
    _abi.rope(**{**ROPE, "n_tokens": 0, "q": None, "positions": None})
    _abi.rope_append(**{**APPEND, "n_tokens": 0, "k": None})
    _abi.rmsnorm_rows(**{**NORM, "rows": 0, "x": None})
    _abi.rmsnorm_rows(**{**NORM, "cols": 0, "y": None})
    _abi.logprobs_rows(**{**LOGPROBS, "rows": 0, "x": None})


CHUNK = dict(dtype=_abi.BF16, cache_type=_abi.BF16, n_rows=4, n_tokens=30, q_heads=4, kv_heads=2, head_dim=64, q=P, ldq=256, starts=2 * P,
             k_pages=3 * P, v_pages=4 * P, num_pages=10, page_size=16, page_stride=2048, tables=5 * P, ld_table=3, lengths=6 * P, o=7 * P,
             ldo=256, scale=0.125, workspace=8 * P, workspace_bytes=1 << 30)


def test_chunk_refused():
    f = _abi.paged_attn_chunk
    for change in (dict(dtype=_abi.F32), dict(cache_type=_abi.F16), dict(head_dim=264, ldq=2000, ldo=2000),
                   dict(head_dim=72, cache_type=_abi.F8E4M3, ldq=2000, ldo=2000, page_stride=1 << 20)):
        refused("UnsupportedBackend", f, **{**CHUNK, **change})
    for change in (dict(n_rows=-1), dict(n_tokens=-1), dict(n_tokens=2 ** 31), dict(q_heads=5), dict(q_heads=0), dict(kv_heads=0), dict(q=None),
                   dict(o=None), dict(starts=None), dict(lengths=None), dict(tables=None), dict(k_pages=None), dict(v_pages=None),
                   dict(ldq=255), dict(ldo=248), dict(ldq=260), dict(q=P + 2), dict(o=7 * P + 8), dict(k_pages=3 * P + 8), dict(page_size=24),
                   dict(page_stride=2047), dict(num_pages=-1), dict(ld_table=-1), dict(window=-1), dict(sinks=-1), dict(o=P), dict(o=P + 256),
                   dict(scale=float("nan")), dict(scale=float("inf")), dict(k_scale=float("inf")), dict(ld_table=1 << 26),
                   dict(n_rows=1 << 22, ld_table=500, page_size=65536, page_stride=1 << 24)):
        refused("Shape", f, **{**CHUNK, **change})
    f(**{**CHUNK, "n_tokens": 0, "q": None})
    f(**{**CHUNK, "n_rows": 0, "starts": None})
    refused("Shape", _abi.paged_attn_chunk_workspace, 1, -1, 4, 2, 64)
    refused("Shape", _abi.paged_attn_chunk_workspace, 1, 1, 5, 2, 64)
