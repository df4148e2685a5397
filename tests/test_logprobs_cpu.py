"""token_logprobs: what the entry point refuses on the host, before any CUDA call."""
import pytest
import torch

from util import pkg

EINVAL, EALIGN, ELIMIT = 1, 3, 5
PTR = 1 << 20                                               # an address that is never read


@pytest.mark.parametrize('change,code', [
    (dict(x=None), EINVAL), (dict(dtype=2), EINVAL), (dict(ld=99), EINVAL), (dict(M=0), EINVAL), (dict(V=0), EINVAL), (dict(G=-1), EINVAL),
    (dict(tokens=None), EINVAL), (dict(lp=None), EINVAL), (dict(ent=None), EINVAL), (dict(top=-1), EINVAL), (dict(ids=None), EINVAL), (dict(tlp=None), EINVAL),
    (dict(V=5, top=6), EINVAL), (dict(top=33), ELIMIT), (dict(M=(1 << 24) + 1), ELIMIT), (dict(V=(1 << 30) + 1, ld=1 << 31), ELIMIT),
    (dict(x=PTR + 2), EALIGN), (dict(x=PTR + 1, dtype=1), EALIGN), (dict(tokens=PTR + 2), EALIGN), (dict(lp=PTR + 1), EALIGN), (dict(ent=PTR + 2), EALIGN),
    (dict(ids=PTR + 3), EALIGN), (dict(tlp=PTR + 2), EALIGN)])
def test_refuses(change, code):
    a = dict(x=PTR, dtype=0, ld=100, M=4, V=100, tokens=PTR, G=1, lp=PTR, ent=PTR, top=5, ids=PTR, tlp=PTR)
    a.update(change)
    assert pkg().lib().b200_token_logprobs(a['x'], a['dtype'], a['ld'], a['M'], a['V'], a['tokens'], a['G'], a['lp'], a['ent'], a['top'], a['ids'],
                                           a['tlp'], None) == code


def test_binding_refuses():
    P = pkg()
    x, t = torch.zeros(4, 100), torch.zeros((4, 1), dtype=torch.int32)
    for bad in ((x[0], t), (x.half(), t), (x.T, t), (x, t[:3]), (x, t.long()), (x, t[:, 0]), (x, torch.zeros((2, 4), dtype=torch.int32).T)):
        with pytest.raises(P.B200Error):
            P.token_logprobs(*bad)
    with pytest.raises(P.B200Error):
        P.token_logprobs(x, t, 2, out=P.token_logprobs_out(t, 3))
    with pytest.raises(P.B200Error, match='current CUDA device'):
        P.token_logprobs(x, t)


def test_clusters_meet_before_they_touch_each_other():
    """Shared memory of another CTA of a cluster may be touched only once that CTA is known to have started: in every kernel a barrier
    of the whole cluster comes before the first address in another CTA's memory."""
    import glob
    import os
    import re
    import __graft_entry__ as G
    seen = 0
    for path in glob.glob(os.path.join(G.PKG_DIR, 'csrc', '*.cu')):
        code = re.sub(r'//[^\n]*', '', open(path).read())
        for kernel in re.split(r'\b__global__\b', code)[1:]:
            kernel = re.split(r'\n}', kernel)[0]                                       # up to the kernel's last line
            remote = re.search(r'map_shared_rank|mapa\(', kernel)
            if remote:
                seen += 1
                assert re.search(r'\w*cluster\w*(\.sync|_wait|\.barrier_wait)\(', kernel[:remote.start()]), (path, kernel[:200])
    assert seen >= 3
