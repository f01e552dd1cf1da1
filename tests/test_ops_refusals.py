"""The operators on row tables and score rows refuse, before anything touches a GPU, calls whose sizes or pointers do
not fit: through the C ABI with made-up addresses that no kernel may see, and through vectordb_amd.ops with CPU tensors."""

import ctypes as C

import pytest
import torch

from vectordb_amd import _native, ops

P = C.c_void_p(4096)        # never dereferenced: every call below is refused on the host


def refused(fn, *args, text):
    lib = _native.load()
    assert getattr(lib, fn)(*args) == _native.VDB_ERR_INVALID
    assert text in _native.last_error(), _native.last_error()


LOOKUP = dict(table=P, tt=0, n_rows=100, dim=8, ld=8, rows=P, n=5, scale=1.0, out=P, ot=0, ldo=8, stream=None)
GRAD = dict(grad=P, gt=0, ld=8, rows=P, n=5, scale=1.0, out=P, ot=0, n_rows=100, dim=8, ldo=8, acc=0, work=P, size=1 << 30, stream=None)
DISTILL = dict(scores=P, t=0, n=4, vocab=50, ld=50, teacher=P, rows=P, k=3, ldt=3, ldr=3, lse=None, tau=1.0, loss=P, stats=P, work=P,
               size=1 << 20, stream=None)
DGRAD = dict(scores=P, t=0, n=4, vocab=50, ld=50, teacher=P, rows=P, k=3, ldt=3, ldr=3, lse=None, tau=1.0, stats=P, gl=P, grad=C.c_void_p(8192),
             ldg=50, stream=None)
STEP = dict(scores=P, t=0, n=4, vocab=50, ld=50, teacher=P, rows=P, k=3, ldt=3, ldr=3, lse=None, tau=1.0, gl=P, loss=P, stats=None,
            grad=C.c_void_p(8192), ldg=50, work=P, size=1 << 20, stream=None)
SAMPLE = dict(scores=P, t=0, n=4, vocab=50, ld=50, sf=0, u=P, dt=None, tau=1.0, dk=None, k=0, dp=None, p=1.0, dm=None, m=0.0, mask=None, mld=0,
              out=P, logp=P, work=P, size=1 << 20, stream=None)


@pytest.mark.parametrize("fn,base,change,text", [
    ("vdb_lookup_dev", LOOKUP, dict(tt=3), "value type"), ("vdb_lookup_dev", LOOKUP, dict(ot=-1), "value type"),
    ("vdb_lookup_dev", LOOKUP, dict(n=-1), "bad sizes"), ("vdb_lookup_dev", LOOKUP, dict(dim=0), "bad sizes"),
    ("vdb_lookup_dev", LOOKUP, dict(n_rows=1 << 31), "bad sizes"), ("vdb_lookup_dev", LOOKUP, dict(ldo=7), "bad sizes"),
    ("vdb_lookup_dev", LOOKUP, dict(ld=-8), "bad sizes"), ("vdb_lookup_dev", LOOKUP, dict(rows=None), "null pointer"),
    ("vdb_lookup_dev", LOOKUP, dict(table=None), "null pointer"), ("vdb_lookup_dev", LOOKUP, dict(out=None), "null pointer"),
    ("vdb_lookup_grad_dev", GRAD, dict(gt=9), "value type"), ("vdb_lookup_grad_dev", GRAD, dict(dim=0), "bad sizes"),
    ("vdb_lookup_grad_dev", GRAD, dict(n=1 << 31), "bad sizes"), ("vdb_lookup_grad_dev", GRAD, dict(ldo=4), "leading dimensions"),
    ("vdb_lookup_grad_dev", GRAD, dict(ld=-1), "leading dimensions"), ("vdb_lookup_grad_dev", GRAD, dict(grad=None), "null pointer"),
    ("vdb_lookup_grad_dev", GRAD, dict(out=None), "null pointer"), ("vdb_lookup_grad_dev", GRAD, dict(n=500, size=16), "workspace"),
    ("vdb_lookup_grad_dev", GRAD, dict(n=500, work=None), "workspace"),
    ("vdb_distill_dev", DISTILL, dict(t=3), "value type"), ("vdb_distill_dev", DISTILL, dict(vocab=0), "bad sizes"),
    ("vdb_distill_dev", DISTILL, dict(k=_native.DISTILL_MAX_K + 1), "slots"), ("vdb_distill_dev", DISTILL, dict(ldr=-3), "slots"),
    ("vdb_distill_dev", DISTILL, dict(tau=0.0), "temperature"), ("vdb_distill_dev", DISTILL, dict(tau=float("nan")), "temperature"),
    ("vdb_distill_dev", DISTILL, dict(teacher=None), "null pointer"), ("vdb_distill_dev", DISTILL, dict(loss=None), "null pointer"),
    ("vdb_distill_grad_dev", DGRAD, dict(ldg=49), "leading dimension"), ("vdb_distill_grad_dev", DGRAD, dict(stats=None), "null pointer"),
    ("vdb_distill_grad_dev", DGRAD, dict(grad=P, ldg=64), "in place"), ("vdb_distill_grad_dev", DGRAD, dict(tau=-1.0), "temperature"),
    ("vdb_distill_step_dev", STEP, dict(ldg=49), "leading dimension"), ("vdb_distill_step_dev", STEP, dict(grad=None), "null pointer"),
    ("vdb_distill_step_dev", STEP, dict(loss=None), "null pointer"), ("vdb_distill_step_dev", STEP, dict(gl=None), "null pointer"),
    ("vdb_sample_dev", SAMPLE, dict(t=7), "value type"), ("vdb_sample_dev", SAMPLE, dict(vocab=(1 << 24) + 1), "bad sizes"),
    ("vdb_sample_dev", SAMPLE, dict(vocab=0), "bad sizes"), ("vdb_sample_dev", SAMPLE, dict(u=None), "null pointer"),
    ("vdb_sample_dev", SAMPLE, dict(out=None), "null pointer"), ("vdb_sample_dev", SAMPLE, dict(mask=P, mld=1), "mask"),
    ("vdb_sample_dev", SAMPLE, dict(ld=-1), "bad sizes"),
])
def test_c_abi_refuses(fn, base, change, text):
    refused(fn, *{**base, **change}.values(), text=text)


ODD = C.c_void_p(4096 + 8)


@pytest.mark.parametrize("fn,base,change,text", [
    ("vdb_lookup_grad_dev", GRAD, dict(work=ODD), "16 bytes"), ("vdb_distill_dev", DISTILL, dict(work=ODD), "16 bytes"),
    ("vdb_distill_step_dev", STEP, dict(work=ODD), "16 bytes"), ("vdb_sample_dev", SAMPLE, dict(work=ODD), "16 bytes"),
    ("vdb_lookup_grad_dev", GRAD, dict(n=1 << 30), "bad sizes"), ("vdb_lookup_grad_dev", GRAD, dict(n_rows=1 << 30), "bad sizes"),
    ("vdb_lookup_grad_dev", GRAD, dict(dim=(1 << 23) + 1, ldo=1 << 24), "bad sizes"),
])
def test_limits(fn, base, change, text):
    refused(fn, *{**base, **change}.values(), text=text)


def test_workspace_sizes():
    lib = _native.load()
    b = C.c_int64(-1)
    assert lib.vdb_lookup_grad_workspace(0, 10, 4, C.byref(b)) == 0 and b.value >= 0
    assert lib.vdb_lookup_grad_workspace(1000, 10, 4, C.byref(b)) == 0 and b.value >= 1000 * 16
    assert lib.vdb_lookup_grad_workspace(-1, 10, 4, C.byref(b)) == _native.VDB_ERR_INVALID
    assert lib.vdb_lookup_grad_workspace(10, 10, 4, None) == _native.VDB_ERR_INVALID
    assert lib.vdb_distill_workspace(10, 0, C.byref(b)) == _native.VDB_ERR_INVALID
    assert lib.vdb_sample_workspace(10, 1 << 25, C.byref(b)) == _native.VDB_ERR_INVALID


def test_empty_calls_need_no_gpu():
    lib = _native.load()
    assert lib.vdb_lookup_dev(*{**LOOKUP, **dict(n=0, rows=None, out=None)}.values()) == 0
    assert lib.vdb_lookup_grad_dev(*{**GRAD, **dict(n_rows=0, out=None)}.values()) == 0
    assert lib.vdb_distill_dev(*{**DISTILL, **dict(n=0, loss=None, size=0, work=None)}.values()) == 0
    assert lib.vdb_sample_dev(*{**SAMPLE, **dict(n=0, u=None, out=None)}.values()) == 0


def test_ops_refuse_cpu_tensors_and_other_objects():
    x, r, u = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    lists = torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int64)
    for call in (lambda: ops.lookup(x, r), lambda: ops.lookup_grad(x, r, 10), lambda: ops.distill(x, *lists), lambda: ops.sample(x, u),
                 lambda: ops.distill_grad(x, *lists, torch.zeros(4, 2), u), lambda: ops.distill_step(x, *lists, u),
                 lambda: ops.sample(x.numpy(), u)):
        with pytest.raises(ValueError):
            call()
