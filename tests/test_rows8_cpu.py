"""Host side of the 8-bit activation operators and the logits' rules: their
argument checks come before any device work, and their workspaces cover what
the calls ask for."""
import ctypes as C

import pytest

import pywelvet

BIG = dict(ws=16, ws_bytes=1 << 62, status=True)
ROWS = pywelvet.rows8(64, 64, 64)


def refused(st, word=None, code=1):
    assert st.code == code, (st.code, st.message)
    assert word is None or word.encode() in st.message, st.message


def accepted(st):
    """The checks passed: there is no device to run on."""
    if pywelvet.available():
        pytest.skip("accepted arguments would be launched")
    assert st.code == 2 and b"dtype" not in st.message, st.message


def test_rows_are_checked():
    store = lambda rows, n=3, width=60, **kw: pywelvet.rows8_store(1, n, width, 64, rows, status=True, **kw)  # noqa: E731
    refused(pywelvet.rows8_store(4, 3, 60, 64, ROWS, status=True), "dtype", 2)
    refused(pywelvet.rows8_load(9, 3, 60, ROWS, 64, status=True), "dtype", 2)
    for n, width in ((-1, 60), (3, 0), (3, -5), (2 ** 24 + 1, 60), (3, 2 ** 24 + 1)):
        refused(store(ROWS, n, width))
    refused(store(ROWS, x_stride=59))
    refused(store(None), "null rows")
    refused(store(pywelvet.rows8(None, 64, 64)), "null")
    refused(store(pywelvet.rows8(64, 64, None)), "null")
    refused(store(pywelvet.rows8(72, 64, 64)), "16")
    refused(store(pywelvet.rows8(64, 72, 64)), "16")
    refused(store(pywelvet.rows8(64, 48, 64)), "stride")  # 60 values are 64 codes
    refused(store(pywelvet.rows8(64, 64, 66)), "aligned")
    refused(pywelvet.rows8_store(1, 3, 60, 66, ROWS, status=True), "aligned")
    refused(pywelvet.rows8_store(3, 3, 60, 65, ROWS, status=True), "aligned")
    accepted(store(ROWS))
    accepted(store(pywelvet.rows8(None, 64, None), n=0))
    accepted(store(pywelvet.rows8(64, 1 << 40, 64), n=2 ** 24))


def test_swiglu_is_checked():
    call = lambda **kw: pywelvet.rows8_swiglu(1, 3, 60, 64, 64, status=True, **kw)  # noqa: E731
    refused(call())
    refused(call(d_h=64, h_stride=59))
    refused(call(d_h=64, gate_stride=59))
    refused(call(d_h=64, up_stride=10))
    refused(call(gate=pywelvet.rows8(64, 32, 64)), "stride")
    refused(call(h=pywelvet.rows8(64, 64, None)), "null")
    refused(pywelvet.rows8_swiglu(2, 3, 60, 65, 64, d_h=64, status=True), "aligned")
    refused(pywelvet.rows8_swiglu(5, 3, 60, 64, 64, d_h=64, status=True), "dtype", 2)
    accepted(call(up=ROWS))
    back = lambda dg=128, du=192, **kw: pywelvet.rows8_swiglu_backward(  # noqa: E731
        1, 3, 60, ROWS, ROWS, 64, dg, du, status=True, **kw)
    refused(pywelvet.rows8_swiglu_backward(1, 3, 60, None, ROWS, 64, 128, 192, status=True), "null rows")
    refused(back(du=128))
    refused(back(dg=None))
    refused(back(dg=64, dgate_stride=61), "stride")
    refused(back(du=64, dup_stride=61), "stride")
    accepted(back(dg=64))
    accepted(back(du=64))


def test_backward_is_checked():
    call = lambda act=-1, dtype=1, n=3, inn=50, out=60, d_dy=64, **kw: pywelvet.rows8_backward(  # noqa: E731
        act, dtype, n, inn, out, d_dy, **{**BIG, **kw})
    refused(call(dtype=4, d_dpre=128), "dtype", 2)
    refused(call())
    for act in (-2, 7, 100):
        refused(call(act=act, pre=ROWS, d_dpre=128), "activation")
    refused(call(act=1, d_dpre=128), "pre-activations")
    refused(call(act=1, pre=pywelvet.rows8(64, 48, 64), d_dpre=128), "stride")
    refused(call(d_dw=128), "rows")
    refused(call(d_dw=128, x=pywelvet.rows8(64, 48, 64)), "stride")
    refused(call(d_dx=128), "layer")
    refused(call(d_dw=130, x=ROWS), "aligned")
    refused(call(d_dpre=64, dpre_stride=61), "dy")
    refused(call(d_dw=128, x=ROWS, ws_bytes=100), "workspace")
    refused(call(d_dw=128, x=ROWS, ws=None), "workspace")
    refused(call(d_dw=128, x=ROWS, ws=24), "workspace")
    refused(call(dy_stride=59, d_dpre=128))
    for n, inn, out in ((-1, 50, 60), (3, 0, 60), (3, 50, 2 ** 20 + 1), (2 ** 20 + 1, 50, 60),
                        (2 ** 20, 50, 2 ** 15 + 2)):  # the last: 2^22 blocks and more
        refused(call(n=n, inn=inn, out=out, d_dpre=128))
        assert pywelvet.lib().welvet_hip_rows8_backward_bytes(1, n, inn, out, C.byref(C.c_size_t())).code == 1
    accepted(call(d_dpre=128, ws=None, ws_bytes=0))
    accepted(call(d_dpre=64))
    accepted(call(d_dw=128, x=ROWS))
    accepted(call(act=6, pre=ROWS, d_dw=128, x=ROWS))


@pytest.mark.parametrize("dtype", [1, 2, 3])
@pytest.mark.parametrize("inn,out", [(1, 1), (777, 1001), (4096, 11008)])
def test_backward_workspace_serves_smaller_batches(dtype, inn, out):
    sizes = [pywelvet.rows8_backward_bytes(dtype, n, inn, out) for n in (*range(0, 300), 2047, 2048, 2049, 8192)]
    assert sizes == sorted(sizes)


def test_layers_are_checked():
    L, h = pywelvet.lib(), C.c_void_p(5)
    f = (C.c_float * 4)(1, 2, 3, 4)
    mount = lambda inn, out, W=f, bias=None, k=0, to=C.byref(h): L.welvet_hip_int8_mount(  # noqa: E731
        inn, out, -1, W, bias, k, to)
    refused(mount(2, 2, to=None))
    for inn, out in ((0, 2), (2, 0), (131073, 1), (1, 2 ** 24 + 1), (131072, 16385)):
        refused(mount(inn, out))
        assert h.value is None
    refused(mount(2, 2, W=None))
    refused(mount(2, 2, k=1))
    refused(L.welvet_hip_int8_mount_device(2, 2, -1, 40, None, 0, C.byref(h)))  # 16-byte aligned
    codes = (C.c_int8 * 4)(1, -127, -128, 0)
    refused(L.welvet_hip_int8_mount_codes(2, 2, -1, codes, f, None, 0, C.byref(h)), "-128")
    refused(L.welvet_hip_int8_mount_codes(2, 2, -1, None, f, None, 0, C.byref(h)))
    refused(L.welvet_hip_int8_mount_dense(None, C.byref(h)))
    refused(L.welvet_hip_int8_mount_dense(None, None))
    refused(L.welvet_hip_int8_bytes(None, 1, C.byref(C.c_size_t())))
    refused(L.welvet_hip_int8_weights(None, None, None))
    refused(L.welvet_hip_int8_forward(None, 1, 1, 64, 64, None, 64, 64, None, 0, 64, 1 << 20, None))
    refused(L.welvet_hip_int8_product(None, 1, 1, C.byref(ROWS), 64, 64, None, 0, 64, 1 << 20, None))
    L.welvet_hip_int8_release(None)
    accepted(mount(2, 2))


def test_rules_are_checked():
    call = lambda dtype=1, n=2, vocab=100, d=64, to=128, stride=None, out_stride=None, mask_stride=None, **kw: \
        pywelvet.LogitRules(mask_stride=mask_stride, **kw).apply(  # noqa: E731
            dtype, n, vocab, d, to, stride=stride, out_stride=out_stride, status=True)
    refused(call(dtype=4), "dtype", 2)
    for n, vocab in ((-1, 100), (2 ** 20 + 1, 100), (2, 0), (2, 2 ** 30 + 1), (2 ** 20, 2 ** 18)):
        refused(call(n=n, vocab=vocab))
    refused(call(d=None))
    refused(call(to=None))
    refused(call(stride=99), "stride")
    refused(call(out_stride=99), "stride")
    refused(call(to=64, out_stride=101), "stride")
    refused(call(d=66), "aligned")
    refused(call(history=5), "rules")
    refused(call(history=5, d_history=64, history_stride=4), "rules")
    refused(call(history=2 ** 20, d_history=64), "rules")
    refused(call(history=-1), "rules")
    refused(call(history=5, d_history=66), "aligned")
    refused(call(biases=3, d_bias=64), "rules")
    refused(call(biases=1025, d_bias=64, d_bias_index=64), "rules")
    refused(call(masks=1), "rules")
    refused(call(masks=1, d_masks=64, mask_stride=3), "rules")
    refused(call(masks=-1, d_masks=64), "rules")
    refused(call(d_frequency=65), "aligned")
    refused(pywelvet.lib().welvet_hip_logits_rules(1, 2, 100, 64, 100, None, 128, 100, None))
    accepted(call())
    accepted(call(n=1, to=64, out_stride=101))
    accepted(call(history=5, d_history=64, biases=1024, d_bias=64, d_bias_index=64, masks=2, d_masks=64))
