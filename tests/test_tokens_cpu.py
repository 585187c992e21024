"""Host side of the token-side operators: their argument checks come before
any device work, and their workspaces cover what the calls ask for."""
import ctypes as C

import pytest

import pywelvet


def test_refused_before_the_device():
    L = pywelvet.lib()
    assert pywelvet.embedding_forward(9, 4, 4, 16, 16, 1, 16, status=True).code == 2
    assert pywelvet.embedding_forward(1, 0, 4, 16, 16, 1, 16, status=True).code == 1
    assert L.welvet_hip_embedding_store_forward(None, 16, 1, 1.0, 16, 4, None).code == 1
    assert pywelvet.embedding_backward(4, 4, 16, 1, None, 16, status=True).code == 1
    st = pywelvet.embedding_backward(4, 4, 16, 300, 16, 16, status=True)
    assert st.code == 1 and b"workspace" in st.message
    a = pywelvet.Adapters(1, 1, 4, 8, 8, 16, 16)
    st = a.forward(16, 16, 3, 16, 16, status=True)
    assert st.code == 1 and b"workspace" in st.message
    assert a.backward(16, 16, 3, 16, 16, status=True).code == 1
    assert L.welvet_hip_adapters_forward(None, 16, 8, 16, 1, None, 0, 16, 8, None, None, 0, None).code == 1
    assert pywelvet.distill(1, 1, 8, 16, 1, 16, 16, d_loss=16, temperature=0.0, status=True).code == 1
    assert pywelvet.distill(7, 1, 8, 16, 1, 16, 16, d_loss=16, status=True).code == 2


def test_no_device_is_unsupported():
    if pywelvet.available():
        pytest.skip("a GPU is present")
    assert pywelvet.embedding_forward(1, 4, 4, 16, 16, 1, 16, status=True).code == 2
    assert pywelvet.distill(1, 1, 8, 16, 1, 16, 16, d_loss=16, status=True).code == 2


def test_sizes_past_a_launch_are_refused():
    b = C.c_size_t()
    L = pywelvet.lib()
    assert L.welvet_hip_embedding_backward_bytes(2**31 - 1, 64, 1, C.byref(b)).code == 1
    assert L.welvet_hip_embedding_backward_bytes(2**31 - 2, 8192, 1, C.byref(b)).code == 1
    assert L.welvet_hip_embedding_backward_bytes(10, 10, 1, None).code == 1
    assert L.welvet_hip_distill_bytes(1, 1, 2**31 - 1, 1, C.byref(b)).code == 1
    a = pywelvet.Adapters(1, 1, 4, 8, 8, 16, 16)
    assert L.welvet_hip_adapters_bytes(a._ref, 2**24 + 1, C.byref(b)).code == 1


@pytest.mark.parametrize("n", [0, 1, 256, 257, 4096, 4097, 100000])
def test_embedding_workspace(n):
    """Nothing up to 256 tokens; above, the order (twice that past 4096 tokens)
    and two partial rows for every 32 tokens."""
    got = pywelvet.embedding_backward_bytes(5000, 100, n)
    if n <= 256:
        assert got == 0
    else:
        assert got >= n * 4 * (4 if n > 4096 else 2) + -(-n // 32) * 2 * 100 * 4


def test_temperatures_without_an_exponent_are_refused():
    """log2(e) / T has to be a float: below some 4.24e-39 it is not, though 1 / T is."""
    call = lambda T: pywelvet.distill(1, 1, 8, 16, 1, 16, 16, d_loss=16, temperature=T, status=True)  # noqa: E731
    for T in (3e-39, 4.2e-39):
        st = call(T)
        assert st.code == 1 and b"temperature" in st.message


def test_gradient_in_place_needs_the_logits_stride():
    """Rows of another stride would be written over rows not yet read."""
    call = lambda n, dstride: pywelvet.distill(  # noqa: E731
        1, n, 8, 16, 1, 16, 16, d_dlogits=16, logits_stride=8, dlogits_stride=dstride, ws=16, ws_bytes=1 << 20,
        status=True)
    st = call(2, 9)
    assert st.code == 1 and b"stride" in st.message
    if not pywelvet.available():  # accepted: then there is no device
        assert call(1, 9).code == 2 and call(2, 8).code == 2


@pytest.mark.parametrize("vocab", [2**31 - 1, 2**31 - 65, 2**31 - 70, 2**31 - 512, 2**31 - 4095])
def test_vocabularies_past_an_int_are_refused(vocab):
    """A block's steps along a row (up to 512 values past its end) are counted in int."""
    b = C.c_size_t()
    for n in (1, 300):
        assert pywelvet.lib().welvet_hip_distill_bytes(3, n, vocab, 1, C.byref(b)).code == 1
        assert pywelvet.distill(3, n, vocab, 16, 1, 16, 16, d_loss=16, ws=16, ws_bytes=1 << 30, status=True).code == 1


def test_distill_workspace_of_the_largest_vocabulary():
    assert pywelvet.distill_bytes(3, 1, 2**31 - 4096, 1) >= 512 * 8 + 4


def embedding_codes(vocab, dim, n):
    """Codes of the lookup, the gradient's workspace and the gradient."""
    b = C.c_size_t()
    return (pywelvet.embedding_forward(1, vocab, dim, 16, 16, n, 16, status=True).code,
            pywelvet.lib().welvet_hip_embedding_backward_bytes(vocab, dim, n, C.byref(b)).code,
            pywelvet.embedding_backward(vocab, dim, 16, n, 16, 16, ws=16, ws_bytes=1 << 62, status=True).code)


@pytest.mark.parametrize("vocab,dim,n,lookup,gradient", [
    (100, 256, 2**26 - 16, True, True),
    (100, 256, 2**26 - 15, True, False),    # the order's 64 threads a row reach 2^32
    (100, 256, 2**26, True, False),
    (100, 256, 2**27, True, False),
    (100, 257, 2**27, False, False),        # 2^25 blocks of 128 threads
    (100, 512, 2**27 - 4, True, False),
    (100, 512, 2**27 - 3, False, False),
    (100, 1024, 2**26 - 64, True, True),
    (100, 1025, 2**26 - 64, False, False),  # two tiles of columns
    (2**25, 1024, 300, True, True),
    (1, 2**31 - 4096, 1, True, True),
    (1, 2**31 - 4096, 3, True, True),
    (1, 2**31 - 4096, 16, True, False),     # up to 256 tokens: one a block
    (1, 2**31 - 4095, 1, False, False),     # a thread's steps along a row pass an int
    (1, 2**31 - 1, 1, False, False),
    (1000, 2**31 - 1000, 2**27, False, False)])
def test_launches_past_32_bits_are_refused(vocab, dim, n, lookup, gradient):
    """What a launch cannot take is code 1 before anything is enqueued."""
    codes = embedding_codes(vocab, dim, n) if not pywelvet.available() else None
    if codes is None:
        pytest.skip("accepted sizes would be launched")
    assert codes == (2 if lookup else 1, 0 if gradient else 1, 2 if gradient else 1)


def test_adapters_launches_past_32_bits_are_refused():
    """The rows' launch: 256 threads for 16 rows and 256 columns; of rows one by
    one the gradients' blocks, counted in int."""
    b = C.c_size_t()

    def codes(count, rank, inn, out, n):
        a = pywelvet.Adapters(1, count, rank, inn, out, 16, 16)
        on = dict(ws=16, ws_bytes=1 << 62, status=True)
        return (pywelvet.lib().welvet_hip_adapters_bytes(a._ref, n, C.byref(b)).code,
                a.forward(16, 16, n, None, 16, **on).code,
                a.backward(16, 16, n, None, 16, d_dx=16, **on).code,
                a.backward(16, 16, n, 16, 16, d_ddown=16, d_dup=16, **on).code)
    if pywelvet.available():
        pytest.skip("accepted sizes would be launched")
    assert codes(1, 1, 64, 8192 - 256, 2**23) == (0, 2, 2, 2)
    assert codes(1, 1, 64, 8192, 2**23) == (0, 1, 2, 2)  # 2^24 blocks
    assert codes(1, 1, 8191, 64, 2**23) == (0, 2, 1, 2)
    assert codes(60000, 1, 2**24, 2**24, 1) == (0, 2, 2, 1)
    assert codes(4, 1, 2**24, 2**24, 1) == (0, 2, 2, 2)


def test_adapters_workspace_of_another_dtype_is_unsupported():
    b = C.c_size_t()
    for dtype in (0, 4, 33):
        a = pywelvet.Adapters(dtype, 1, 4, 8, 8, 16, 16)
        assert pywelvet.lib().welvet_hip_adapters_bytes(a._ref, 4, C.byref(b)).code == 2


def accepted(st):
    """The checks passed: the call ran, or there is no device to run it on."""
    return st.code != 1


@pytest.mark.parametrize("dtype,vocab,k", [(1, 32000, 20), (3, 131072, 64), (2, 50257, 1024), (1, 2047, 5), (3, 5000, 1)])
def test_distill_workspace_serves_smaller_batches(dtype, vocab, k):
    """A workspace sized for n rows is enough for every smaller batch, on both
    sides of the 256 rows from which a row has one block and needs none."""
    sizes = [pywelvet.distill_bytes(dtype, n, vocab, k) for n in range(0, 600)]
    assert sizes == sorted(sizes)
    assert pywelvet.distill_bytes(dtype, 1 << 22, vocab, k) == sizes[-1]
    if pywelvet.available():
        return
    for n in range(1, 300):
        assert accepted(pywelvet.distill(dtype, n, vocab, 16, k, 16, 16, d_loss=16, ws=16, ws_bytes=sizes[-1],
                                         status=True))


@pytest.mark.parametrize("dtype,count,rank,inn,out", [
    (3, 8, 16, 4096, 4096), (2, 4, 64, 4096, 4096), (3, 8, 32, 4096, 11008), (1, 1, 8, 2048, 8192),
    (1, 3, 5, 1001, 777), (3, 2, 256, 8192, 64), (1, 5, 1, 1, 1), (2, 4, 130, 515, 20000)])
def test_adapters_workspace_serves_smaller_batches(dtype, count, rank, inn, out):
    """A workspace sized for n rows is enough for every smaller batch in both
    directions, where rows go one by one and where they are sorted into blocks
    whose length grows with n."""
    a = pywelvet.Adapters(dtype, count, rank, inn, out, 16, 16)
    ns = sorted({*range(0, 2100, 7), *(2 ** i + d for i in range(20) for d in (-1, 0, 1, 9)),
                 *range(2040, 2060), *(16 * i + d for i in range(1, 130) for d in (0, 1))})
    sizes = [a.workspace_bytes(n) for n in ns]
    assert sizes == sorted(sizes)
    if pywelvet.available():
        return
    for most in (130, 2049, 8192):
        on = dict(ws=16, ws_bytes=a.workspace_bytes(most), status=True)
        for n in (n for n in ns if 0 < n <= most):
            assert accepted(a.forward(16, 16, n, None, 16, **on)), (n, most)
            assert accepted(a.backward(16, 16, n, 16, 16, d_dx=16, d_ddown=16, d_dup=16, **on)), (n, most)


@pytest.mark.parametrize("n", [257, 2047, 2048, 2049, 4096, 4097, 65536, 65537, 600001])
def test_embedding_workspace_by_chunks(n):
    """The order's two arrays, four past one chunk of 2048 tokens, and two
    partial rows for every 32 tokens; not less for more tokens."""
    got = pywelvet.embedding_backward_bytes(5000, 100, n)
    assert got >= n * 4 * (4 if n > 2048 else 2) + -(-n // 32) * 2 * 100 * 4
    assert got <= pywelvet.embedding_backward_bytes(5000, 100, n + 1)
