"""What the losses on rows of raw predictions refuse (no GPU needed: arguments are looked at before any device)."""
import pytest
import torch

from tests.conftest import has_gpu

Z = 4096    # an address that is never read


def _distill(lib, **kw):
    a = dict(device=0, stream=None, z=Z, dtype=0, n=4, K=5, ldz=5, ids=Z, t=Z, tdtype=0, T=2, tail=0, w=None, tau=1.0, loss=Z, g=Z, ldg=5, h=None, ldh=5, work=None)
    a.update(kw)
    return lib.evb_distill_grads(*a.values())


def _policy(lib, **kw):
    a = dict(device=0, stream=None, z=Z, dtype=0, n=4, K=5, ldz=5, action=Z, old=Z, adv=Z, ref=None, w=None, tau=1.0, lo=0.2, hi=0.2, beta=0.0, loss=Z,
             logp=Z, g=Z, ldg=5, h=None, ldh=5)
    a.update(kw)
    return lib.evb_policy_grads(*a.values())


def _preference(lib, **kw):
    a = dict(device=0, stream=None, z=Z, dtype=0, n=4, K=5, ldz=5, label=Z, seq=Z, pairs=1, ref=None, w=None, beta=0.1, smooth=0.0, mean=0, loss=Z,
             margin=Z, logp=Z, g=Z, ldg=5, work=Z)
    a.update(kw)
    return lib.evb_preference_grads(*a.values())


NAN = float("nan")
ROWS = [dict(dtype=1), dict(dtype=2), dict(dtype=9), dict(n=-1), dict(n=2_000_000_001), dict(K=0, ldz=0), dict(ldz=4), dict(ldg=4), dict(z=None), dict(z=Z + 2),
        dict(g=Z + 1, dtype=3)]


@pytest.mark.parametrize("kw", ROWS + [dict(T=0), dict(tdtype=1), dict(tau=0.0), dict(tau=-1.0), dict(tau=NAN), dict(tau=float("inf")), dict(tail=1, tau=2.0),
                                       dict(ids=None), dict(t=None), dict(h=Z, ldh=4), dict(h=Z + 2), dict(work=Z + 8)])
def test_distill_refuses(pkg, kw):
    from evotrees_b200 import _lib
    assert _distill(_lib.lib(), **kw) == -1 and b"evb_distill_grads" in _lib.lib().evb_last_error()


@pytest.mark.parametrize("kw", ROWS + [dict(tau=0.0), dict(tau=NAN), dict(lo=-0.1), dict(lo=1.5), dict(hi=-1.0), dict(hi=NAN), dict(beta=-1.0), dict(beta=NAN),
                                       dict(action=None), dict(old=None), dict(adv=None)])
def test_policy_refuses(pkg, kw):
    from evotrees_b200 import _lib
    assert _policy(_lib.lib(), **kw) == -1 and b"evb_policy_grads" in _lib.lib().evb_last_error()


@pytest.mark.parametrize("kw", ROWS + [dict(pairs=-1), dict(beta=-0.1), dict(beta=NAN), dict(smooth=1.5), dict(smooth=NAN), dict(label=None), dict(seq=None),
                                       dict(loss=None), dict(margin=None), dict(logp=None), dict(work=None), dict(work=Z + 4)])
def test_preference_refuses(pkg, kw):
    from evotrees_b200 import _lib
    assert _preference(_lib.lib(), **kw) == -1 and b"evb_preference_grads" in _lib.lib().evb_last_error()


def test_limits(pkg):
    from evotrees_b200 import _lib
    lib = _lib.lib()
    big = (1 << 20) + 1
    assert _distill(lib, K=big, ldz=big, ldg=big) == -7 and b"1048576" in lib.evb_last_error()
    assert _policy(lib, K=big, ldz=big, ldg=big) == -7 and _preference(lib, K=big, ldz=big, ldg=big) == -7
    assert _distill(lib, T=1025) == -7 and b"1024" in lib.evb_last_error()


@pytest.mark.skipif(has_gpu(), reason="checks the behaviour of a machine without a GPU")
def test_no_gpu_fails_loudly(pkg):
    from evotrees_b200 import _lib
    for f in (_distill, _policy, _preference):
        assert f(_lib.lib()) == -2 and b"no CPU fallback" in _lib.lib().evb_last_error()


def test_python_refuses(pkg):
    z, i, f = torch.zeros((4, 5)), torch.ones(4, dtype=torch.int32), torch.zeros(4)
    with pytest.raises(pkg.EvbError, match="no CPU fallback"):
        pkg.policy_grads(z, i, f, f)
    for bad in (z.double(), z[0], z.long(), z.numpy()):
        with pytest.raises(ValueError, match="`pred`"):
            pkg.distill_grads(bad, i[:, None], f[:, None])
    with pytest.raises(AttributeError):
        pkg.no_such_name


@pytest.mark.gpu
def test_python_refuses_on_gpu(pkg):
    z, i, f = torch.zeros((4, 5), device="cuda"), torch.ones(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    seq = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    ok = lambda **kw: pkg.policy_grads(**{**dict(pred=z, action=i, old_logp=f, adv=f), **kw})       # noqa: E731
    ok()
    for kw in (dict(pred=z.t()), dict(pred=z[:, ::2]), dict(pred=z[:1].expand(4, 5)), dict(pred=z[:, :0]), dict(action=i.long()), dict(action=i[:3]),
               dict(action=i.cpu()), dict(old_logp=f.double()), dict(adv=f[::2]), dict(adv=torch.zeros(8, device="cuda")[::2]), dict(w=f[:2]),
               dict(ref_logp=f.half()), dict(adv=None)):
        with pytest.raises(ValueError):
            ok(**kw)
    for kw in (dict(clip=(2.0, 0.2)), dict(tau=0.0), dict(beta=-1.0)):
        with pytest.raises(pkg.EvbError, match="evb -1"):
            ok(**kw)
    with pytest.raises(ValueError, match="`ids`"):
        pkg.distill_grads(z, i, f)
    with pytest.raises(ValueError, match="`teacher`"):
        pkg.distill_grads(z, i[:, None], i[:, None])
    with pytest.raises(ValueError, match="`teacher`"):
        pkg.distill_grads(z, i[:, None], f[:2, None])
    with pytest.raises(ValueError, match="`seq`"):
        pkg.preference_grads(z, i, seq[:2])
    with pytest.raises(ValueError, match="`seq`"):
        pkg.preference_grads(z, i, seq.long())
    with pytest.raises(ValueError, match="`w`"):
        pkg.preference_grads(z, i, seq, w=f)
    with pytest.raises(pkg.EvbError):
        pkg.distill_grads(z, i[:, None], f[:, None], tail=True, tau=2.0)
