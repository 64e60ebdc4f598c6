"""Scalar-quantised rows: arguments that the C ABI refuses before anything runs
on a device, and the sizes it reports (no GPU).  The addresses are never read:
every call here is refused, or has no rows."""
import pytest

import insitu_b200 as ib

P = 1 << 20          # an address of any alignment asked for
OK, EINVAL = 0, -1


def lib():
    return ib.load_library(require_device=False)


WRITE = dict(x=P, x_type=0, n=4, d=32, ldx=32, slots=P, bits=8, group=0, codes=P, ldc=32, scales=P, lds=1,
             capacity=16, claim=None, stream=None)
READ = dict(codes=P, ldc=32, scales=P, lds=1, capacity=16, bits=8, group=0, slots=P, n=4, d=32, out=P, out_type=0,
            ldo=32, stream=None)
MATMUL = dict(a=P, lda=32, a_scale=P, m=4, b=P, ldb=32, b_scale=P, n=8, k=32, bias=None, out=P, out_type=0, ldo=8,
              work=None, work_bytes=0, stream=None)
SCORES = dict(x=P, x_type=0, ldx=32, m=8, codes=P, ldc=32, scales=P, n=8, d=32, bias=None, out=P, out_type=0, ldo=8,
              work=P, work_bytes=1 << 20, stream=None)


def call(name, base, **change):
    L = lib()
    rc = getattr(L, name)(*{**base, **change}.values())
    return rc, L.ivf_global_last_error().decode()


@pytest.mark.parametrize("change", [
    dict(x_type=3), dict(x_type=-1), dict(n=-1), dict(n=1 << 31), dict(d=0), dict(d=(1 << 20) + 1), dict(ldx=31),
    dict(x=None), dict(x=P + 2), dict(x_type=1, x=P + 1), dict(bits=2), dict(bits=16), dict(group=-16),
    dict(group=8), dict(group=24), dict(codes=None), dict(scales=None), dict(scales=P + 2), dict(ldc=31),
    dict(bits=4, ldc=15), dict(group=16, lds=1), dict(capacity=-1), dict(capacity=1 << 31),
    dict(slots=None, n=17), dict(slots=P + 4), dict(ldx=1 << 32), dict(n=513, capacity=1000, claim=None), dict(n=513, capacity=1000, claim=P + 2)])
def test_write_refuses(change):
    rc, msg = call("ivf_sq_write", WRITE, **change)
    assert rc == EINVAL and msg


@pytest.mark.parametrize("change", [
    dict(out_type=3), dict(n=-1), dict(n=1 << 31), dict(d=0), dict(d=(1 << 20) + 1), dict(ldo=31), dict(out=None),
    dict(out=P + 2), dict(bits=1), dict(group=40), dict(codes=None), dict(scales=None), dict(ldc=31),
    dict(group=16, lds=1), dict(capacity=-1), dict(slots=None, n=17), dict(slots=P + 4)])
def test_read_refuses(change):
    rc, msg = call("ivf_sq_read", READ, **change)
    assert rc == EINVAL and msg


@pytest.mark.parametrize("change", [
    dict(m=-1), dict(m=1 << 31), dict(n=-1), dict(n=1 << 31), dict(k=0), dict(k=131072), dict(lda=31), dict(ldb=31),
    dict(ldo=7), dict(a=None), dict(b=None), dict(a_scale=None), dict(b_scale=None), dict(out=None),
    dict(out_type=7), dict(out=P + 2), dict(out_type=2, out=P + 1), dict(a_scale=P + 1), dict(b_scale=P + 2),
    dict(bias=P + 3), dict(work=P + 8), dict(m=8, a=P + 1), dict(m=8, b=P + 4, work=P, work_bytes=8 * 32 - 1),
    dict(m=8, k=31, lda=31, work=P, work_bytes=8 * 32 - 1)])
def test_matmul_refuses(change):
    rc, msg = call("ivf_sq_matmul", MATMUL, **change)
    assert rc == EINVAL and msg


@pytest.mark.parametrize("change", [
    dict(x_type=3), dict(ldx=31), dict(m=-1), dict(n=-1), dict(d=0), dict(d=131072), dict(ldc=31), dict(ldo=7),
    dict(x=None), dict(codes=None), dict(scales=None), dict(out=None), dict(work=None), dict(work=P + 8),
    dict(work_bytes=8 * 32 + 4 * 8 - 1)])
def test_scores_refuses(change):
    rc, msg = call("ivf_sq_scores", SCORES, **change)
    assert rc == EINVAL and msg


def test_calls_without_rows_do_nothing():
    assert call("ivf_sq_write", WRITE, n=0, x=None)[0] == OK
    assert call("ivf_sq_write", WRITE, capacity=0, codes=None, scales=None)[0] == OK
    assert call("ivf_sq_read", READ, n=0, out=None)[0] == OK
    assert call("ivf_sq_matmul", MATMUL, m=0, a=None, a_scale=None, out=None)[0] == OK
    assert call("ivf_sq_matmul", MATMUL, n=0, b=None, b_scale=None, out=None)[0] == OK
    assert call("ivf_sq_scores", SCORES, m=0, x=None, out=None)[0] == OK
    assert call("ivf_sq_scores", SCORES, n=0, codes=None, scales=None, out=None)[0] == OK


def test_scratch_sizes():
    L = lib()

    def scores(m, d, codes=P, ldc=None, n=50):
        return L.ivf_sq_scores_work(m, codes, ldc or (d + 15) // 16 * 16, n, d)

    matmul = L.ivf_sq_matmul_work
    assert scores(10, 96) >= 10 * (96 + 4)
    assert scores(10, 97) >= 10 * (112 + 4)
    assert scores(10, 96, codes=P + 1) >= 10 * (96 + 4) + 50 * 96          # a store whose rows are copied first
    assert scores(10, 97, ldc=97) >= 10 * (112 + 4) + 50 * 112
    assert scores((1 << 31) - 2, 131071) >= ((1 << 31) - 2) * (131072 + 4)
    assert scores(1, 96) == scores(0, 96) == scores(10, 96, n=0) == 0      # nothing to keep between two kernels
    assert scores(-1, 8) == scores(8, 0) == scores(8, 131072) == scores(10, 96, ldc=95) == 0
    assert matmul(P, 48, 10, P, 64, 20, 33) == 0
    assert matmul(P + 1, 48, 10, P, 64, 20, 33) == 10 * 48
    assert matmul(P, 48, 10, P, 33, 20, 33) == 20 * 48
    assert matmul(P, 33, 10, P, 33, 20, 33) == 30 * 48
    assert matmul(P, 33, 1, P, 33, 20, 33) == matmul(P, 33, 0, P, 33, 20, 33) == matmul(P, 32, 10, P, 33, 20, 33) == 0


def test_binding_refuses_without_a_device():
    import torch

    with pytest.raises(ValueError):          # not CUDA tensors
        a = torch.zeros(2, 8, dtype=torch.int8)
        ib.sq_matmul(a, torch.ones(2), a, torch.ones(2))
    with pytest.raises(ValueError):          # not int8
        a = torch.zeros(2, 8)
        ib.sq_matmul(a, torch.ones(2), a, torch.ones(2))
    if not torch.cuda.is_available():
        with pytest.raises(RuntimeError):
            ib.SQRows(8, 8)
