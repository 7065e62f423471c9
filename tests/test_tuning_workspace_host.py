"""Workspaces are refused when they are missing, too small or off their alignment: at the C entries, before any device work."""
import ctypes

from memintelli_flash_b200 import _native as N

FAKE = ctypes.c_void_p(0x1000)          # never dereferenced: every call below fails its host checks


def _rows(**kw):
    f = dict(logits=0x1000, targets=0x1000, cu_seqlens=None, rows=4, cols=8, layout=N.OutLayout(4, 0, 8, 1),
             ignore_index=-100, sequences=2, rows_per_sequence=2, temperature=1.0, dtype=N.F32, targets_i64=1, cu_i64=1,
             reserved=0)
    f.update(kw)
    return N.TokenRows(**f)


def _entries():
    """Each entry as a function of its workspace and the workspace's bytes."""
    L, lay = N.lib(), N.OutLayout(4, 0, 8, 1)
    one, types, numel = (N.c_vp * 1)(0x1000), (N.c_i32 * 1)(N.F32), (N.c_i64 * 1)(4)
    policy = N.PolicySpec(0.2, 0.2, 0.0, 0, 0)
    pref = N.PreferenceSpec(0.1, 0.0, 0.0, 0, 0)
    yield lambda ws, n: L.mib_policy_loss(_rows(), policy, FAKE, FAKE, None, FAKE, FAKE, FAKE, lay, ws, n, None)
    yield lambda ws, n: L.mib_preference_loss(_rows(), pref, None, FAKE, FAKE, FAKE, FAKE, FAKE, lay, ws, n, None)
    yield lambda ws, n: L.mib_loss_grad(_rows(), ws, n, None, FAKE, lay, None)
    yield lambda ws, n: L.mib_embedding_grad(FAKE, 1, 4, FAKE, N.F32, 8, 9, 8, 1.0, -1, FAKE, N.F32, 8, 0, ws, n, None)
    yield lambda ws, n: L.mib_clip_grad_norm(one, one, numel, types, types, 1, 2, 1.0, 1e-6, FAKE, ws, n, None)


def test_workspaces_are_checked():
    for entry in _entries():
        for ws, n, word in ((None, 1 << 30, b"missing"), (FAKE, 16, b"too small"), (FAKE, 0, b"too small"),
                            (ctypes.c_void_p(0x1080), 1 << 30, b"256-byte"), (ctypes.c_void_p(0x1001), 1 << 30, b"256-byte")):
            assert entry(ws, n) == N.MIB_ERR_PARAM and word in N.lib().mib_last_error()


def test_loss_grad_arguments_are_checked():
    L, lay = N.lib(), N.OutLayout(4, 0, 8, 1)
    call = lambda rows=None, factor=None, grad=FAKE, lay=lay: L.mib_loss_grad(rows or _rows(), FAKE, 1 << 30, factor, grad, lay, None)  # noqa: E731
    assert call(_rows(logits=None)) == N.MIB_ERR_PARAM
    assert call(_rows(dtype=9)) == N.MIB_ERR_UNSUPPORTED
    assert call(_rows(sequences=-1)) == N.MIB_ERR_SHAPE
    assert call(grad=None) == N.MIB_ERR_PARAM
    assert call(grad=ctypes.c_void_p(0x1002)) == N.MIB_ERR_PARAM
    assert call(factor=ctypes.c_void_p(0x1002)) == N.MIB_ERR_PARAM
    assert call(lay=N.OutLayout(4, 0, 7, 1)) == N.MIB_ERR_SHAPE
    assert call(lay=N.OutLayout(4, 0, 8, 2)) == N.MIB_ERR_SHAPE
