"""Scalar-quantised rows whose values are so small that 1 / scale leaves fp32's
range: their zeros have the code 0 in every alignment."""
import numpy as np
import pytest
import torch

import insitu_b200 as ib
from test_gpu_sq import check_write, new_store, ref_quantise

pytestmark = pytest.mark.gpu


def tiny_rows(d, t):
    """rows with zeros among values of 127 * 2^-120 down to the type's smallest"""
    v = []
    for e in (-120, -125, -126, -127, -128, -129, -130, -135, -142):
        r = np.zeros(d)
        r[0], r[1], r[-1] = 127 * 2.0 ** e, -3.4 * 2.0 ** e, 63.5 * 2.0 ** e
        v.append(r)
    r = np.zeros(d)
    r[d // 2] = 2.0 ** -133                              # the smallest bf16
    v += [r, -r, np.zeros(d)]
    return torch.from_numpy(np.array(v)).to(t).cuda()


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("d,group,pad,offset", [(33, 0, 0, 0), (64, 16, 0, 0), (33, 0, 1, 0), (64, 16, 1, 0),
                                                (64, 0, 0, 3), (3000, 0, 1, 0)])
def test_zeros_of_tiny_rows(cuda_ok, t, bits, d, group, pad, offset):
    x = tiny_rows(d, t)
    rows, buf = new_store(x.shape[0], d, bits, group, pad, offset)
    check_write(rows, buf, x, None, offset)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [33, 64])
@pytest.mark.parametrize("m", [1, 3, 12])
def test_scores_of_tiny_rows(cuda_ok, t, d, m):
    """against unit vectors the scores are the query's codes times its scale and 127 times theirs"""
    x = tiny_rows(d, t).roll(-6, 0)[:m]                  # from 127 * 2^-130 on
    store = ib.SQRows(d, d).write(torch.eye(d, device="cuda"))
    codes, scale = ref_quantise(x, 8, 0)
    got = store.scores(x).cpu().numpy()
    assert ((got == 0) == (codes == 0)).all()
    q = ib.SQRows(m, d).write(x)
    assert np.array_equal(q.codes[:, :d].cpu().numpy(), codes)
    assert np.array_equal(got, ib.sq_matmul(q.codes[:, :d], q.scales[:, 0], store.codes[:, :d],
                                            store.scales[:, 0]).cpu().numpy())
