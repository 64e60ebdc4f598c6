"""Scalar-quantised rows on the GPU (ivf_sq_write, ivf_sq_read, ivf_sq_matmul,
ivf_sq_scores) against their definition in 64 bits.

Codes, scales and 8-bit sums are compared for equality: their definition leaves
no freedom (the scale is the fp32 quotient, the code the rounded quotient by
that scale, the sum is whole).  Tolerances, with u = 2^-24 (half a step of fp32)
and h = eps / 2 of the output type:
  read    value = code * scale: one fp32 product (u), then the type's rounding
          (h): |error| <= (u + h) |value|, plus half the type's smallest number
  matmul  float(sum) (u), * a_scale (u), then one fused multiply-add with the
          bias (u of the result), then the type's rounding (h):
          |error| <= 2 u (1 + u) |sum * sa * sb| + (u + h (1 + u)) |y'| + tiny, where |y'| is
          at most |y| plus the first term
"""
import numpy as np
import pytest
import torch

import insitu_b200 as ib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def tiny(t):
    fi = torch.finfo(t)
    return fi.tiny * fi.eps / 2          # half the smallest subnormal


def groups_of(d, group):
    return -(-d // group) if group else 1


def ref_quantise(x, bits, group):
    """(codes int64 [n, d], scales fp32 [n, groups]) of x (a float tensor), on the CPU in 64 bits"""
    v = x.double().cpu().numpy()
    n, d = v.shape
    L = 127 if bits == 8 else 7
    G, w = groups_of(d, group), group or d
    codes, scales = np.zeros((n, d), np.int64), np.zeros((n, G), np.float32)
    for g in range(G):
        part = v[:, g * w:(g + 1) * w]
        with np.errstate(all="ignore"):
            amax = np.abs(part).max(1)                       # NaN wins, then infinity
            s = (amax.astype(np.float32) / np.float32(L)).astype(np.float32)
            s = np.where(np.isnan(part).any(1), np.float32(np.nan), s)
            ok = np.isfinite(s) & (s > 0)
            q = np.rint(part / np.where(ok, s.astype(np.float64), 1.0)[:, None])
        codes[:, g * w:(g + 1) * w] = np.where(ok[:, None], np.clip(q, -L, L), 0)
        scales[:, g] = s
    return codes, scales


def pack(codes, bits):
    if bits == 8:
        return codes.astype(np.int8).view(np.uint8)
    c = np.zeros((codes.shape[0], (codes.shape[1] + 1) // 2 * 2), np.int64)
    c[:, :codes.shape[1]] = codes
    return ((c[:, 0::2] & 15) | ((c[:, 1::2] & 15) << 4)).astype(np.uint8)


def new_store(capacity, d, bits, group, pad=0, offset=0, fill=0x5a):
    """a store whose bytes are all known: rows of the least length rounded up to 16, plus pad, from byte `offset`"""
    rb = (d * bits + 7) // 8
    ld = (rb + 15) // 16 * 16 + pad
    buf = torch.full((capacity * ld + offset + 16,), fill, dtype=torch.uint8, device="cuda")
    codes = buf[offset:offset + capacity * ld].view(capacity, ld)
    if bits == 8:
        codes = codes.view(torch.int8)
    scales = torch.full((capacity, groups_of(d, group)), -5.0, device="cuda")
    return ib.SQRows.from_arrays(codes, scales, d, bits, group), buf


def ref_store(buf, scales0, rows, x, slots, offset=0):
    """the bytes of buf and the scales after the write, by the definition"""
    b = buf.cpu().numpy().copy()
    s = scales0.copy()
    codes, sc = ref_quantise(x, rows.bits, rows.group)
    by = pack(codes, rows.bits)
    ld = rows._ldc
    for i, t in enumerate(slots):
        if 0 <= t < rows.capacity:
            b[offset + t * ld:offset + t * ld + by.shape[1]] = by[i]
            s[t] = sc[i]
    return b, s


def rows_of(n, d, t, seed, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, d, generator=g, device="cuda") * torch.exp(spread * torch.randn(n, 1, generator=g, device="cuda"))
    if n > 2:
        x[1] = 0
    return x.to(t)


def check_write(rows, buf, x, slots, offset=0):
    before, s0 = buf.clone(), rows.scales.cpu().numpy().copy()
    rows.write(x, None if slots is None else torch.tensor(slots, dtype=torch.int64, device="cuda"))
    exp_b, exp_s = ref_store(before, s0, rows, x, range(x.shape[0]) if slots is None else slots, offset)
    assert np.array_equal(rows.scales.cpu().numpy().view(np.uint32)[~np.isnan(exp_s)],
                          exp_s.view(np.uint32)[~np.isnan(exp_s)])
    assert np.array_equal(np.isnan(rows.scales.cpu().numpy()), np.isnan(exp_s))
    assert np.array_equal(buf.cpu().numpy(), exp_b)


SHAPES = [(1, 0), (2, 0), (7, 0), (16, 16), (17, 16), (33, 32), (96, 32), (127, 0), (128, 0), (128, 64), (129, 128),
          (257, 0), (300, 64), (1000, 64), (1024, 0), (1031, 0), (2047, 0), (4097, 0), (9001, 0), (9001, 2048)]


@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("t", TYPES)
def test_write_read(cuda_ok, d, group, bits, t):
    n, cap = 37, 41
    rows, buf = new_store(cap, d, bits, group)
    x = rows_of(n, d, t, d + bits)
    slots = np.random.default_rng(d).permutation(cap)[:n].tolist()
    check_write(rows, buf, x, slots)
    rows2, buf2 = new_store(cap, d, bits, group)
    check_write(rows2, buf2, x, None)
    # read back, every type; a slot outside reads as zeros
    codes, sc = ref_quantise(x, bits, group)
    w = group or d
    val = codes * np.repeat(sc.astype(np.float64), w, axis=1)[:, :d]
    at = torch.tensor(slots + [-1, cap, 1 << 40], device="cuda")
    for o in TYPES:
        got = rows.read(at, dtype=o)
        assert (got[n:] == 0).all() and got.dtype == o
        err = np.abs(got[:n].double().cpu().numpy() - val)
        assert (err <= (U + half(o)) * np.abs(val) + tiny(o)).all()
    assert torch.equal(rows2.read(torch.arange(n, device="cuda"), dtype=t), rows.read(at[:n], dtype=t))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d,group,pad,offset,skip,step", [(96, 0, 1, 0, 0, 96), (96, 32, 0, 3, 0, 100),
                                                          (130, 0, 0, 0, 1, 133), (128, 64, 8, 8, 3, 160),
                                                          (500, 0, 2, 2, 1, 501), (2500, 0, 4, 4, 1, 2501)])
def test_write_read_unaligned(cuda_ok, bits, t, d, group, pad, offset, skip, step):
    n, cap = 19, 23
    wide = rows_of(n, step + skip, t, 77 + d)
    x = wide[:, skip:skip + d]
    rows, buf = new_store(cap, d, bits, group, pad, offset)
    slots = np.random.default_rng(5).permutation(cap)[:n].tolist()
    check_write(rows, buf, x, slots, offset)
    ref, b2 = new_store(cap, d, bits, group)
    ref.write(x.contiguous(), torch.tensor(slots, device="cuda"))
    at = torch.tensor(slots, device="cuda")
    out = torch.full((n, d + 5), 7.0, dtype=t, device="cuda")
    rows.read(at, out=out[:, 3:3 + d])
    assert torch.equal(out[:, 3:3 + d], ref.read(at, dtype=t))
    assert (out[:, :3] == 7).all() and (out[:, 3 + d:] == 7).all()


@pytest.mark.parametrize("n", [1, 2, 64, 511, 512, 513, 3000])
@pytest.mark.parametrize("d,group", [(40, 0), (40, 16), (700, 0), (9000, 0)])
def test_write_repeated_and_outside_slots(cuda_ok, n, d, group):
    """of rows with one slot the last stays whole; rows outside the store are left out"""
    if n * d > 5_000_000:
        n = 600
    cap = max(3, n // 3)
    rows, buf = new_store(cap, d, 8, group)
    x = rows_of(n, d, torch.float32, n)
    g = np.random.default_rng(n)
    slots = g.integers(-2, cap + 2, n)
    slots[g.random(n) < 0.2] = 1
    if n > 4:
        slots[0], slots[-1] = -(1 << 40), 1 << 40
    check_write(rows, buf, x, slots.tolist())


def test_write_ties_and_extremes(cuda_ok):
    inf, nan = float("inf"), float("nan")
    top = 3.3895313892515355e38
    v = []
    for amax in (127.0, 254.0, 381.0, 127 * 2.0 ** -90, 127 * 2.0 ** -99, 127 * 2.0 ** -100, 127 * 2.0 ** -101,
                 127 * 2.0 ** -126, 127 * 2.0 ** -149, 100 * 2.0 ** -149, 2.0 ** -149, 64 * 2.0 ** -149, top, 1.0,
                 0.1, 3.0, 126.99999, 127.00001):
        s = np.float32(np.float32(amax) / np.float32(127))
        r = np.zeros(256, np.float32)
        b = (np.arange(-127, 127) + 0.5).astype(np.float64) * np.float64(s)    # the borders between codes
        r[:254] = b.astype(np.float32)
        r[255] = amax
        v.append(r)
        v.append(np.nextafter(r, np.float32(0)))
        v.append(np.where(np.arange(256) < 254, np.nextafter(r, np.float32(np.inf)), r).astype(np.float32))
    v = np.array(v, np.float32)
    x = torch.from_numpy(np.clip(v, -top, top)).cuda()
    rows, buf = new_store(x.shape[0], 256, 8, 0)
    check_write(rows, buf, x, None)
    rows, buf = new_store(x.shape[0], 256, 4, 32)
    check_write(rows, buf, x, None)
    # NaN and infinities poison their group alone
    y = torch.randn(5, 64, device="cuda")
    y[0, 3], y[1, 40], y[2, 0], y[3] = nan, inf, -inf, -0.0
    y[4, 1], y[4, 2] = inf, nan
    for t in TYPES:
        rows, buf = new_store(5, 64, 8, 32)
        check_write(rows, buf, y.to(t), None)
        got = rows.read(dtype=t)
        bad = torch.isnan(got)
        exp = torch.zeros(5, 64, dtype=torch.bool, device="cuda")
        exp[0, :32] = exp[1, 32:] = exp[2, :32] = exp[4, :32] = True
        assert torch.equal(bad, exp) and (got[3] == 0).all()


def test_long_offsets(cuda_ok):
    """a store and an output whose bytes pass 2^32"""
    cap, d = 34_000_000, 128
    codes = torch.empty(cap, d, dtype=torch.int8, device="cuda")
    scales = torch.empty(cap, 1, device="cuda")
    rows = ib.SQRows.from_arrays(codes, scales, d)
    n = 1000
    x = rows_of(n, d, torch.float32, 3)
    slots = torch.arange(cap - n, cap, device="cuda")
    rows.write(x, slots)
    c, s = ref_quantise(x, 8, 0)
    assert np.array_equal(codes[cap - n:].cpu().numpy(), c)
    assert np.array_equal(scales[cap - n:].cpu().numpy(), s)
    big = torch.empty(cap // 2, d, dtype=torch.float32, device="cuda")       # 8.7 GB
    at = torch.full((cap // 2,), cap - 1, device="cuda")
    at[-n:] = slots
    rows.read(at, out=big)
    assert torch.equal(big[-n:], rows.read(slots)) and torch.equal(big[12345], rows.read(slots[-1:])[0])
    del big, at
    # the product over the end of the store
    q = rows_of(3, d, torch.float32, 4)
    tail = ib.SQRows.from_arrays(codes[cap - n:], scales[cap - n:], d)
    exp = tail.scores(q)
    few = ib.SQRows.from_arrays(codes, scales, d).scores(q, dtype=torch.bfloat16)
    assert torch.equal(few[:, cap - n:], exp.bfloat16())


# ---------------------------------------------------------------------------
# the product
# ---------------------------------------------------------------------------

def codes_of(n, k, seed, ld=None, offset=0, full=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = ld or k
    buf = torch.randint(-128, 128, (n * ld + offset,), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    return buf[offset:offset + n * ld].view(n, ld)[:, :k]


def scales_of(n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.exp(torch.randn(n, generator=g, device="cuda")) * 1e-3


def check_product(got, a, sa, b, sb, bias, t):
    """got against the 64-bit product (sums below 2^53: exact in double)"""
    acc = a.double() @ b.double().t()
    p = acc * sa.double()[:, None] * sb.double()
    y = p if bias is None else p + bias.double()
    first = 2 * U * (1 + U) * p.abs()
    tol = first + (U + half(t) * (1 + U)) * (y.abs() + first) + tiny(t)
    err = (got.double() - y).abs()
    assert got.dtype == t and got.shape == y.shape
    assert (err <= tol).all(), (float((err / (y.abs() + 1e-30)).max()), int((err > tol).sum()))


SIZES = [(1, 1, 1), (1, 5, 3), (1, 300, 128), (2, 77, 96), (3, 1000, 256), (4, 129, 4096), (5, 65, 16), (7, 2, 8193),
         (8, 640, 130), (9, 640, 131), (15, 33, 64), (16, 257, 1024), (17, 128, 128), (31, 1000, 100), (32, 7, 2000),
         (33, 4096, 32), (64, 64, 64), (65, 65, 65), (100, 1, 500), (128, 128, 128), (129, 300, 129), (255, 255, 255),
         (257, 513, 384), (300, 1000, 1031), (1000, 3, 77), (513, 1025, 2048)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(cuda_ok, m, n, k):
    sa, sb = scales_of(m, 1), scales_of(n, 2)
    bias = torch.randn(n, device="cuda")
    for ld, off in (((k + 15) // 16 * 16, 0), (k, 0), (k + 3, 1)):
        a, b = codes_of(m, k, m + k, ld, off), codes_of(n, k, n + k + 1, ld, off)
        for t in TYPES:
            check_product(ib.sq_matmul(a, sa, b, sb, dtype=t), a, sa, b, sb, None, t)
        check_product(ib.sq_matmul(a, sa, b, sb, bias=bias), a, sa, b, sb, bias, torch.float32)


@pytest.mark.parametrize("m,n", [(1, 9), (2, 200), (20, 130), (130, 300)])
def test_matmul_largest_sums(cuda_ok, m, n):
    """the longest k with every product at its largest: 131071 * 2^14 < 2^31"""
    k = 131071
    for ld in (131072, 131071):
        a = torch.full((m, ld), -128, dtype=torch.int8, device="cuda")[:, :k]
        b = torch.full((n, ld), -128, dtype=torch.int8, device="cuda")[:, :k]
        one = torch.ones(max(m, n), device="cuda")
        got = ib.sq_matmul(a, one[:m], b, one[:n])
        assert (got == float(np.float32(k * 16384))).all()


@pytest.mark.parametrize("m", [1, 6, 16, 40, 200])
def test_matmul_output_rows_and_bad_scales(cuda_ok, m):
    """a wide output's other columns stay; a NaN or infinite scale marks its row or column alone"""
    n, k = 333, 160
    a, b = codes_of(m, k, 1), codes_of(n, k, 2)
    sa, sb = scales_of(m, 3), scales_of(n, 4)
    for t in TYPES:
        for lo, ld in ((0, 352), (5, 341)):
            out = torch.full((m, ld), 3.0, dtype=t, device="cuda")
            ib.sq_matmul(a, sa, b, sb, out=out[:, lo:lo + n])
            check_product(out[:, lo:lo + n], a, sa, b, sb, None, t)
            assert (out[:, :lo] == 3).all() and (out[:, lo + n:] == 3).all()
    sa[m // 2], sb[7] = float("nan"), float("nan")
    got = torch.isnan(ib.sq_matmul(a, sa, b, sb))
    assert got[m // 2].all() and got[:, 7].all()
    got[m // 2], got[:, 7] = False, False
    assert not got.any()


@pytest.mark.parametrize("m,n,d", [(1, 1000, 128), (1, 300, 4096), (2, 77, 96), (4, 129, 1031), (8, 500, 130), (9, 500, 128),
                                   (33, 1000, 96), (200, 2000, 128), (300, 257, 1000), (3, 40, 20000),
                                   (3, 300001, 128)])
@pytest.mark.parametrize("t", TYPES)
def test_scores(cuda_ok, m, n, d, t):
    """equal to the product of the rows as write quantises them"""
    store = ib.SQRows(n, d).write(rows_of(n, d, torch.float32, 8))
    x = rows_of(m, d, t, 9)
    q = ib.SQRows(m, d).write(x)
    bias = torch.randn(n, device="cuda")
    wide = torch.zeros(m, d + 3, dtype=t, device="cuda")
    wide[:, 1:1 + d] = x
    for o in TYPES:
        got = store.scores(x, dtype=o, bias=bias)
        check_product(got, q.codes[:, :d], q.scales[:, 0], store.codes[:, :d], store.scales[:, 0], bias, o)
        assert torch.equal(got, ib.sq_matmul(q.codes[:, :d], q.scales[:, 0], store.codes[:, :d],
                                             store.scales[:, 0], bias=bias, dtype=o))
        assert torch.equal(got, store.scores(wide[:, 1:1 + d], dtype=o, bias=bias))


@pytest.mark.parametrize("m", [1, 3, 9, 40, 300])
@pytest.mark.parametrize("d,pad,offset", [(100, 1, 0), (128, 0, 5), (33, 0, 8)])
def test_scores_of_an_unaligned_store(cuda_ok, m, d, pad, offset):
    n = 259
    rows, _ = new_store(n, d, 8, 0, pad, offset)
    x = rows_of(n, d, torch.float32, 4)
    ref = ib.SQRows(n, d).write(x)
    rows.write(x)
    q = rows_of(m, d, torch.bfloat16, 5)
    assert torch.equal(rows.scores(q), ref.scores(q))
    assert torch.equal(rows.scores(q, dtype=torch.float16), ref.scores(q, dtype=torch.float16))


def test_run_together(cuda_ok):
    """rows inserted, replaced, scored and read back: the best rows are the true neighbours, and rescoring the
    candidates with their values ranks them as the scores do"""
    cap, d, nq = 5000, 96, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    base = torch.nn.functional.normalize(torch.randn(cap, d, generator=g, device="cuda"))
    q = torch.nn.functional.normalize(base[::cap // nq][:nq] + 0.03 * torch.randn(nq, d, generator=g, device="cuda"))
    store = ib.SQRows(cap, d)
    order = torch.randperm(cap, generator=g, device="cuda")
    store.write(torch.randn(cap, d, generator=g, device="cuda"))     # all replaced below
    for part in order.split(700):
        store.write(base[part], part)
    s = store.scores(q)
    # scores differ from the true products by the two roundings: |code error| <= scale / 2 a value
    best = s.argmax(1)
    assert torch.equal(best, (q.double() @ base.double().t()).argmax(1))
    top = s.topk(20, dim=1).indices
    cand = store.read(top.reshape(-1)).view(nq, 20, d)
    qq = ib.SQRows(nq, d).write(q).read()
    again = torch.einsum("qd,qkd->qk", qq.double(), cand.double())
    ref = s.gather(1, top).double()
    # read: u a value; product: 4 u of the sum's terms
    tol = 8 * U * torch.einsum("qd,qkd->qk", qq.double().abs(), cand.double().abs())
    assert ((again - ref).abs() <= tol).all()


def test_graph_and_streams(cuda_ok):
    """captured and replayed on new inputs; on a stream of its own; two captured graphs that run at once"""
    d, n, m = 128, 700, 40
    store = ib.SQRows(2000, d)
    x, slots = rows_of(n, d, torch.bfloat16, 1), torch.randperm(2000, device="cuda")[:n]
    q = [rows_of(m, d, torch.float32, 2), rows_of(3, d, torch.float32, 3)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        store.write(x, slots)
        warm = [store.scores(v) for v in q]
        store.read(slots)
    torch.cuda.synchronize()
    g1, g2, g3 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        store.write(x, slots)
        back = store.read(slots)
    with torch.cuda.graph(g2):
        y2 = store.scores(q[0])
    with torch.cuda.graph(g3):
        y3 = store.scores(q[1])
    x.copy_(rows_of(n, d, torch.bfloat16, 11))
    q[0].copy_(rows_of(m, d, torch.float32, 12))
    q[1].copy_(rows_of(3, d, torch.float32, 13))
    g1.replay()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(s1):
            g2.replay()
        with torch.cuda.stream(s2):
            g3.replay()
    torch.cuda.synchronize()
    ref = ib.SQRows(n, d).write(x)
    assert torch.equal(back, ref.read())
    assert torch.equal(y2, store.scores(q[0])) and torch.equal(y3, store.scores(q[1]))
    assert not torch.equal(y2, warm[0])


def test_write_scratch_outlives_the_store(cuda_ok):
    """a large write on another stream than the first one's, the store dropped while it waits: its scratch is
    not handed out to others before it has run"""
    n, cap = 2000, 1 << 20
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(n, 32, generator=gen).cuda()
    slots = torch.randint(0, cap, (n,), generator=gen).cuda()
    codes = torch.zeros(cap, 32, dtype=torch.int8, device="cuda")
    scales = torch.zeros(cap, 1, device="cuda")
    rows = ib.SQRows.from_arrays(codes, scales, 32)
    rows.write(x, slots)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        rows.write(x, slots)
    del rows
    others = [torch.full((cap,), -7, dtype=torch.int32, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    for o in others:
        assert bool((o == -7).all())


def test_captured_write_outlives_the_store(cuda_ok):
    """a graph of a large write, replayed after its store is gone: the scratch is the graph's own"""
    n, cap = 2000, 1 << 20
    gen = torch.Generator().manual_seed(6)
    x = torch.randn(n, 32, generator=gen).cuda()
    slots = torch.randint(0, cap, (n,), generator=gen).cuda()
    codes = torch.zeros(cap, 32, dtype=torch.int8, device="cuda")
    scales = torch.zeros(cap, 1, device="cuda")
    rows = ib.SQRows.from_arrays(codes, scales, 32)
    rows.write(x, slots)
    want = codes.clone(), scales.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows.write(x, slots)
    del rows
    codes.zero_()
    scales.zero_()
    others = [torch.full((cap,), -7, dtype=torch.int32, device="cuda") for _ in range(4)]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
    for o in others:
        assert bool((o == -7).all())


def test_binding_refusals(cuda_ok):
    store = ib.SQRows(10, 32)
    x = torch.randn(4, 32, device="cuda")
    for bad in (x[:, :31], x.double(), x.cpu(), x[0]):
        with pytest.raises(ValueError):
            store.write(bad)
        with pytest.raises(ValueError):
            store.scores(bad)
    with pytest.raises(ValueError):
        store.write(torch.randn(11, 32, device="cuda"))
    with pytest.raises(ValueError):
        store.write(x, torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        store.write(x, torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError):
        store.read(out=torch.empty(10, 31, device="cuda"))
    with pytest.raises(ValueError):
        store.read(out=torch.empty(32, 10, device="cuda").t())
    with pytest.raises(ValueError):
        store.read(dtype=torch.float64)
    with pytest.raises(ValueError):
        ib.SQRows(10, 32, bits=4).scores(x)
    with pytest.raises(ValueError):
        ib.SQRows(10, 32, group=16).scores(x)
    with pytest.raises(ValueError):
        ib.SQRows(10, 32, group=12)
    with pytest.raises(ValueError):
        ib.SQRows.from_arrays(store.codes, store.scales, 33)
    with pytest.raises(ValueError):
        ib.sq_matmul(store.codes, store.scales[:, 0], store.codes[:, :31], store.scales[:, 0])
    # a transposed or broadcast input is copied, not misread
    t = torch.randn(32, 4, device="cuda").t()
    assert torch.equal(ib.SQRows(4, 32).write(t).read(), ib.SQRows(4, 32).write(t.contiguous()).read())
    e = torch.randn(1, 32, device="cuda").expand(4, 32)
    assert torch.equal(ib.SQRows(4, 32).write(e).read(), ib.SQRows(4, 32).write(e.contiguous()).read())
    # int32 slots, no rows, an empty store
    s32 = torch.tensor([3, 1], dtype=torch.int32, device="cuda")
    store.write(x[:2], s32)
    assert torch.equal(store.read(s32), ib.SQRows(2, 32).write(x[:2]).read())
    assert store.read(s32[:0]).shape == (0, 32) and store.scores(x[:0]).shape == (0, 10)
    store.write(x[:0])
    empty = ib.SQRows(0, 32)
    assert empty.write(x, torch.arange(4, device="cuda")).scores(x).shape == (4, 0)
