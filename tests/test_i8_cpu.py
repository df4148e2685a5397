"""8-bit products: what the entry points refuse on the host, before any CUDA call."""
import ctypes as C

import pytest
import torch

from util import pkg

OK, EINVAL, EALIGN, ELIMIT = 0, 1, 3, 5
PTR = 1 << 20                                               # an address that is never read


def test_pitch_and_workspace():
    L = pkg().lib()
    assert [L.b200_i8_pitch(k) for k in (-1, 0, 1, 32, 17, 4096)] == [0, 0, 32, 32, 32, 4096]
    for M, K in ((1, 1), (5, 2051), (2048, 4096)):
        n = L.b200_i8_gemm_workspace_bytes(M, K)
        assert n % 256 == 0 and n >= M * ((K + 31) // 32 * 32 + 4)
    assert L.b200_i8_gemm_workspace_bytes(1 << 24, 65536) > 1 << 40      # no 32-bit product


@pytest.mark.parametrize('change,code', [
    (dict(x=None), EINVAL), (dict(q=None), EINVAL), (dict(scale=None), EINVAL), (dict(dtype=2), EINVAL), (dict(dtype=-1), EINVAL),
    (dict(ldx=63), EINVAL), (dict(rows=0), EINVAL), (dict(rows=-1), EINVAL), (dict(K=0), EINVAL), (dict(K=65537, ldx=65537), ELIMIT),
    (dict(rows=(1 << 24) + 1), ELIMIT), (dict(x=PTR + 2), EALIGN), (dict(x=PTR + 1, dtype=1), EALIGN), (dict(q=PTR + 8), EALIGN),
    (dict(scale=PTR + 2), EALIGN)])
def test_quantize_refuses(change, code):
    a = dict(x=PTR, dtype=0, ldx=64, rows=4, K=64, q=PTR, scale=PTR)
    a.update(change)
    assert pkg().lib().b200_i8_quantize(a['x'], a['dtype'], a['ldx'], a['rows'], a['K'], a['q'], a['scale'], None) == code


@pytest.mark.parametrize('change,code', [
    (dict(y=None), EINVAL), (dict(x=None), EINVAL), (dict(wq=None), EINVAL), (dict(ws_=None), EINVAL), (dict(ws=None), EINVAL),
    (dict(M=0), EINVAL), (dict(N=0), EINVAL), (dict(K=0), EINVAL), (dict(yd=2), EINVAL), (dict(xd=3), EINVAL), (dict(ldx=63), EINVAL),
    (dict(M=(1 << 24) + 1), ELIMIT), (dict(N=(1 << 24) + 1), ELIMIT), (dict(K=65537, ldx=65537), ELIMIT),
    (dict(y=PTR + 2), EALIGN), (dict(y=PTR + 1, yd=1), EALIGN), (dict(wq=PTR + 8), EALIGN), (dict(ws_=PTR + 1), EALIGN), (dict(ws=PTR + 128), EALIGN),
    (dict(x=PTR + 2), EALIGN)])
def test_gemm_refuses(change, code):
    P = pkg()
    a = dict(y=PTR, yd=0, wq=PTR, ws_=PTR, x=PTR, xd=0, ldx=64, M=4, N=8, K=64, ws=PTR)
    a.update(change)
    W = P.I8RowsC(a['wq'], a['ws_'])
    assert P.lib().b200_i8_gemm(a['y'], a['yd'], C.byref(W), a['x'], a['xd'], a['ldx'], a['M'], a['N'], a['K'], a['ws'], None) == code


@pytest.mark.parametrize('q,scale,code', [(None, PTR, EINVAL), (PTR, None, EINVAL), (PTR + 4, PTR, EALIGN), (PTR, PTR + 3, EALIGN)])
def test_gemm_refuses_rows(q, scale, code):
    P = pkg()
    W, x = P.I8RowsC(PTR, PTR), P.I8RowsC(q, scale)
    assert P.lib().b200_i8_gemm(PTR, 0, C.byref(W), C.addressof(x), P.I8, 0, 4, 8, 64, None, None) == code


def test_binding_refuses():
    P = pkg()
    for bad in (torch.zeros(4), torch.zeros(2, 3, 4), torch.zeros(4, 8, dtype=torch.float16), torch.zeros(8, 4).T, torch.zeros(1, 8).expand(4, 8),
                torch.zeros(0, 8), torch.zeros(4, 0), torch.zeros(4, 16)[:, ::2]):
        with pytest.raises(P.B200Error):
            P.i8_quantize(bad)
    with pytest.raises(P.B200Error, match='current CUDA device'):
        P.i8_quantize(torch.zeros(4, 8))
    with pytest.raises(P.B200Error):
        P.I8Rows(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4), 8)             # rows are 32 bytes apart
    with pytest.raises(P.B200Error):
        P.I8Rows(torch.zeros(4, 32, dtype=torch.int8), torch.zeros(5), 8)
    with pytest.raises(P.B200Error):
        P.I8Rows.empty(0, 8, 'cpu')


def test_binding_keeps_what_it_points_to(monkeypatch):
    """The rows' descriptors are host structures: they have to be alive while the library reads them, temporaries too."""
    import gc
    import importlib
    import weakref
    import __graft_entry__ as G
    P, b = pkg(), importlib.import_module(G.PKG_NAME + '.binding')
    seen = []

    class Fake:
        def b200_i8_gemm(self, *a):
            gc.collect()
            seen.append([r() is not None for r in refs])
            return 0

    monkeypatch.setattr(b, '_device', lambda *t: None)
    monkeypatch.setattr(b, '_stream', lambda s: None)
    monkeypatch.setattr(torch._C, '_cuda_getDevice', lambda: -1, raising=False)      # where CPU tensors say they are
    monkeypatch.setattr(torch._C, '_cuda_getCurrentRawStream', lambda d: 0, raising=False)
    monkeypatch.setattr(b, 'lib', lambda: Fake())
    refs = []

    def rows():
        r = P.I8Rows(torch.zeros((4, 32), dtype=torch.int8), torch.zeros(4), 16)
        refs.append(weakref.ref(r))
        return r

    b.i8_gemm(rows(), rows())
    assert seen == [[True, True]]
    W = rows()
    with pytest.raises(AttributeError):
        W.q = torch.zeros((4, 32), dtype=torch.int8)                                 # the descriptor points to the first one
    with pytest.raises(AttributeError):
        W.scale = torch.ones(4)
    x = torch.zeros(4, 16)
    for ws in (torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(1 << 20, dtype=torch.uint8)[::2], torch.zeros(100, dtype=torch.uint8)):
        with pytest.raises(P.B200Error, match='ws'):
            b.i8_gemm(W, x, ws=ws)


def test_weights_are_read_behind_the_dependency_wait():
    """Only the kernel's own griddepcontrol.wait makes an earlier kernel's writes visible, one that wrote the weights before the call's
    quantiser too: the thread that asks for weights has waited by then, whatever the launch was told."""
    import glob
    import os
    import re
    import __graft_entry__ as G
    source = lambda name: re.sub(r'//[^\n]*', '', open(os.path.join(G.PKG_DIR, 'csrc', name)).read())
    kernels = re.split(r'\b__global__\b', source('gemm_i8.cu'))[1:]
    assert len(kernels) == 2
    for k in kernels:
        start = re.search(r'if \(!p\.early\) pdl_wait\(\);', k)
        loader = k[k.index('if (warp == 0) {'):]
        first = re.search(r'(gx_tma_2d|gi_tma_pair)\([^;]*map_w', loader)
        waited = re.search(r'if \(p\.early\) \{(?:[^{}]|\{[^{}]*\})*pdl_wait\(\);\s*\}', loader)
        assert start and first and waited and waited.end() < first.start()
    gemv = re.split(r'\b__global__\b', source('gemv_i8.cu'))[1]
    wait, first = re.search(r'^    pdl_wait\(\);', gemv, re.M), re.search(r'^ *(if \(.*\) )?load\(wa\);', gemv, re.M)
    assert wait and first and wait.end() < first.start()


def test_the_message_of_a_misaligned_pointer_holds_for_every_call():
    """Codes want 16 bytes, scratch 256: the message of B200_EALIGN names no number."""
    import re
    L = pkg().lib()
    assert 'align' in L.b200_nvfp4_strerror(EALIGN).decode() and not re.search(r'\d', L.b200_nvfp4_strerror(EALIGN).decode())
