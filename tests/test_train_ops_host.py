"""Refusals of the label-loss and AdamW entries that need no GPU: the C ABI's argument checks (before any HIP call), the host-side table of
AdamW, and what the Python wrappers refuse of CPU tensors."""
import ctypes

import numpy as np
import pytest

OK, INVALID, UNSUPPORTED, WORKSPACE = 0, -1, -2, -4


@pytest.fixture(scope="module")
def lib():
    from em_adapt_tensorflow_amd import _lib
    return _lib.load()


def _logp(lib, logits=4096, dtype=0, ldl=24, labels=8192, M=4, C=21, logp=16384, lse=None):
    return lib.emadapt_label_logp(logits, dtype, ldl, labels, M, C, logp, lse, None)


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(M=-1), dict(C=0), dict(ldl=20), dict(logits=None), dict(labels=None), dict(labels=8196),
                                dict(logits=4098), dict(logp=None)])
def test_label_logp_refuses(lib, kw):
    assert _logp(lib, **kw) == INVALID


def test_label_logp_sizes(lib):
    assert _logp(lib, ldl=1 << 31, C=21) == UNSUPPORTED
    assert _logp(lib, M=0, logits=None, labels=None) == OK


def test_label_logp_bwd_refuses(lib):
    def call(logits=1 << 20, lse=1 << 22, dlogp=1 << 23, d=1 << 24, ddt=0, M=4):
        return lib.emadapt_label_logp_bwd(logits, 0, 24, 8192, lse, dlogp, M, 21, d, ddt, None)
    assert call(lse=None) == INVALID and call(dlogp=None) == INVALID and call(d=None) == INVALID
    assert call(ddt=5) == INVALID and call(d=(1 << 24) + 2) == INVALID
    assert call(d=(1 << 20)) == INVALID                      # in place
    assert call(d=(1 << 20) + 4 * 24 * 4 - 4) == INVALID     # the last element shared
    assert call(M=0) == OK


def test_policy_loss_refuses(lib):
    big = 1 << 30

    def call(old=big, ref=None, adv=big, w=None, lo=0.2, hi=0.2, sums=big, logp=big, d=None, M=4, ws=big, nws=1 << 20, kl=0.0):
        return lib.emadapt_policy_loss(1 << 20, 0, 24, 8192, old, ref, adv, w, M, 21, lo, hi, kl, 1.0, sums, logp, d, 0, ws, nws, None)
    for kw in (dict(old=None), dict(adv=None), dict(sums=None), dict(logp=None), dict(lo=-0.1), dict(lo=1.5), dict(hi=-0.1), dict(hi=float("nan")),
               dict(d=1 << 20)):
        assert call(**kw) == INVALID, kw
    assert call(ws=None) == WORKSPACE and call(nws=8) == WORKSPACE and call(ws=big + 4) == WORKSPACE
    assert lib.emadapt_policy_loss_workspace_bytes(1000, 21) > lib.emadapt_policy_loss_workspace_bytes(0, 21) > 0


def test_preference_loss_refuses(lib):
    big = 1 << 30

    def call(at=big, pairs=2, ref=big, smooth=0.0, loss=big, seq=big, d=None, ws=big, nws=1 << 20):
        return lib.emadapt_preference_loss(1 << 20, 0, 24, 8192, at, pairs, ref, 4, 21, 0.1, smooth, 1.0, loss, seq, d, 0, ws, nws, None)
    for kw in (dict(at=None), dict(ref=None), dict(loss=None), dict(seq=None), dict(pairs=-1), dict(smooth=1.5), dict(smooth=float("nan")), dict(at=big + 4),
               dict(d=1 << 20)):
        assert call(**kw) == INVALID, kw
    assert call(ws=None) == WORKSPACE and call(nws=8) == WORKSPACE
    assert call(pairs=1 << 31) == UNSUPPORTED


def _tensor(n, at=0, e=None, wd=0.0, ls=1.0, w=1 << 20, g=1 << 21, m=1 << 22, v=1 << 23):
    from em_adapt_tensorflow_amd._lib import AdamwTensor
    t = AdamwTensor()
    t.w, t.g, t.m, t.v, t.e, t.n, t.unit, t.weight_decay, t.lr_scale = w, g, m, v, e, n, at, wd, ls
    return t


def _table(lib, tensors, gdt=0, state=0, short=0):
    from em_adapt_tensorflow_amd._lib import AdamwTensor
    arr = (AdamwTensor * max(len(tensors), 1))(*tensors)
    chunks = lib.emadapt_adamw_chunks(len(tensors), arr)
    buf = np.zeros(max(lib.emadapt_adamw_table_bytes(max(chunks, 0)) - short, 0) + 64, np.uint8)
    rc = lib.emadapt_adamw_table(len(tensors), arr, gdt, state, buf.ctypes.data, buf.size - 64)
    return rc, chunks, buf


def test_adamw_table_covers_every_element_once(lib):
    sizes = [1, 0, 4096, 4097, 12289, 63]
    at = np.cumsum([0] + [(n + 255) // 256 * 256 for n in sizes])[:-1]
    tensors = [_tensor(n, int(a), e=(1 << 24) + int(a) // 32, wd=0.01 * k, ls=1.0 + k, w=(1 << 26) + 4 * int(a), g=(1 << 28) + 2 * int(a),
                       m=(1 << 22) + int(a), v=(1 << 23) + int(a)) for k, (n, a) in enumerate(zip(sizes, at))]
    rc, chunks, buf = _table(lib, tensors, gdt=1, state=1)
    assert rc == OK
    rec = buf[:chunks * (lib.emadapt_adamw_table_bytes(2) - lib.emadapt_adamw_table_bytes(1))].view(np.dtype([
        ("w", "<u8"), ("g", "<u8"), ("m", "<u8"), ("v", "<u8"), ("e", "<u8"), ("unit", "<u8"), ("n", "<i4"), ("wd", "<f4"), ("ls", "<f4"), ("pad", "<i4")]))
    got = {k: 0 for k in range(len(sizes))}
    for r in rec:
        k = int(np.searchsorted(at, r["unit"], side="right")) - 1
        while sizes[k] == 0:
            k -= 1
        off = int(r["unit"]) - int(at[k])
        assert off == got[k] and r["n"] > 0
        got[k] += int(r["n"])
        t = tensors[k]
        assert (r["w"], r["g"], r["m"], r["v"], r["e"]) == (t.w + 4 * off, t.g + 2 * off, t.m + off, t.v + off, t.e + off // 64 * 2)
        assert off % 64 == 0 and r["wd"] == np.float32(t.weight_decay) and r["ls"] == np.float32(t.lr_scale)
    assert [got[k] for k in range(len(sizes))] == sizes


def test_adamw_table_refuses(lib):
    assert _table(lib, [_tensor(-1)])[1] == INVALID
    assert lib.emadapt_adamw_chunks(2, None) == INVALID and lib.emadapt_adamw_chunks(-1, None) == INVALID
    for kw in (dict(w=0), dict(g=0), dict(m=0), dict(v=0), dict(w=(1 << 20) + 2), dict(g=(1 << 21) + 2)):
        assert _table(lib, [_tensor(5, **kw)])[0] == INVALID, kw
    assert _table(lib, [_tensor(5)], state=1)[0] == INVALID                      # no powers
    assert _table(lib, [_tensor(5, e=1 << 24, m=(1 << 22) + 1)], state=1)[0] == INVALID
    assert _table(lib, [_tensor(5, e=(1 << 24) + 1)], state=1)[0] == INVALID
    assert _table(lib, [_tensor(5)], gdt=2)[0] == INVALID and _table(lib, [_tensor(5)], state=2)[0] == INVALID
    assert _table(lib, [_tensor(5)], short=1)[0] == WORKSPACE
    assert _table(lib, [_tensor(0)])[:2] == (OK, 0)


def test_adamw_step_refuses(lib):
    size = lib.emadapt_adamw_control_bytes()

    def call(table=4096, chunks=1, gdt=0, state=0, ctl=8192, n=size, b1=0.9, b2=0.999, eps=1e-8, max_norm=0.0):
        return lib.emadapt_adamw_step(table, chunks, gdt, state, ctl, n, 1e-3, b1, b2, eps, 1.0, max_norm, 0, 0, None)
    for kw in (dict(table=None), dict(chunks=-1), dict(gdt=3), dict(state=3), dict(b1=1.0), dict(b1=-0.1), dict(b2=1.0), dict(b2=float("nan")), dict(eps=0.0),
               dict(eps=float("nan")), dict(max_norm=-1.0), dict(max_norm=float("nan"))):
        assert call(**kw) == INVALID, kw
    assert call(ctl=None) == WORKSPACE and call(n=size - 1) == WORKSPACE
    assert call(chunks=1 << 31) == UNSUPPORTED


def test_adamw_pack_unpack_refuse(lib):
    assert lib.emadapt_adamw_unpack(4096, 4096, 4096, 63, 4096, 4096, 0, None) == INVALID
    assert lib.emadapt_adamw_unpack(4096, 4096, 4096, 64, None, 4096, 0, None) == INVALID
    assert lib.emadapt_adamw_unpack(4096, 4096, 4096, 64, 4096, 4096, 7, None) == INVALID
    assert lib.emadapt_adamw_pack(4096, 4096, 64, 4096, 4097, 4096, None) == INVALID
    assert lib.emadapt_adamw_pack(4096, 4096, -64, 4096, 4096, 4096, None) == INVALID
    assert lib.emadapt_adamw_unpack(None, None, None, 0, None, None, 0, None) == OK


def test_wrappers_refuse_cpu_tensors():
    import torch
    from em_adapt_tensorflow_amd import ops
    z, lab, f = torch.zeros(4, 24), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    with pytest.raises(ValueError):
        ops.label_logp(z, lab, 21)
    with pytest.raises(ValueError):
        ops.label_logp_bwd(z, lab, f, f, 21)
    with pytest.raises(ValueError):
        ops.policy_loss(z, lab, f, f, 21)
    with pytest.raises(ValueError):
        ops.preference_loss(z, lab, torch.tensor([0, 2, 4]), torch.zeros(2), 21)
    with pytest.raises(ValueError):
        ops.AdamW([torch.zeros(4)], [torch.zeros(4)])
    with pytest.raises(ValueError):
        ops.AdamW([], [])


def test_scalars_that_are_not_finite_are_refused(lib):
    big, size = 1 << 30, lib.emadapt_adamw_control_bytes()
    for bad in (float("nan"), float("inf")):
        for kl, scale in ((bad, 1.0), (0.1, bad)):
            assert lib.emadapt_policy_loss(1 << 20, 0, 24, 8192, big, big, big, None, 4, 21, 0.2, 0.2, kl, scale, big, big, None, 0, big, 1 << 20, None) == INVALID
        for beta, scale in ((bad, 1.0), (0.1, bad)):
            assert lib.emadapt_preference_loss(1 << 20, 0, 24, 8192, big, 2, big, 4, 21, beta, 0.0, scale, big, big, None, 0, big, 1 << 20, None) == INVALID
        for lr, scale in ((bad, 1.0), (1e-3, bad)):
            assert lib.emadapt_adamw_step(4096, 1, 0, 0, 8192, size, lr, 0.9, 0.999, 1e-8, scale, 0.0, 0, 0, None) == INVALID
        assert _table(lib, [_tensor(5, wd=bad)])[0] == INVALID and _table(lib, [_tensor(5, ls=bad)])[0] == INVALID


def test_rows_beyond_any_memory_are_refused(lib):
    assert _logp(lib, ldl=1 << 30, C=21, M=1 << 39) == UNSUPPORTED


def test_tensors_of_two_lists_may_not_share_memory():
    import torch
    from em_adapt_tensorflow_amd import ops
    room = torch.zeros(100)
    a, b = [room[:10], room[40:60]], [room[10:40], room[10:20], room[60:]]
    ops._refuse_shared(a, "params", b, "grads")
    for more in (room[5:6], room[30:41], room[59:61], room):
        with pytest.raises(ValueError, match="share memory"):
            ops._refuse_shared(a, "params", b + [more], "grads")
    ops._refuse_shared(a, "params", b + [room[50:50]], "grads")
