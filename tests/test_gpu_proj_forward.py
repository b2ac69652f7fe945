"""fm_proj_forward: 4-bit projections that share their input, against the product in 64 bits."""
import numpy as np
import pytest
import torch

import moe_ref

pytestmark = pytest.mark.gpu


def context(pkg, host=False, max_batch=64, **kw):
    cfg = pkg.default_config(num_full_layers=0, num_linear_layers=0, max_batch_tokens=max_batch, **kw)
    c = pkg.Context(cfg, host_pointers=host)
    if not host:
        c.set_stream(torch.cuda.current_stream().cuda_stream)
    return c


def on_device(pkg, mat):
    w, s, b = mat
    cuda = lambda a, t: torch.from_numpy(a.view(t)).cuda()  # noqa: E731
    return pkg.proj_weights(cuda(w, np.int32), cuda(s, np.int16).view(torch.bfloat16), cuda(b, np.int16).view(torch.bfloat16))


def run(pkg, c, mats, x):
    xd = torch.from_numpy(np.asarray(x, np.float32)).cuda()
    ys = [torch.full((len(x) + 1, m[0].shape[0]), 7.0, device="cuda") for m in mats]
    c.proj_forward([on_device(pkg, m) for m in mats], len(x), xd, ys)
    c.synchronize()
    for y in ys:
        assert torch.all(y[len(x):] == 7.0)  # rows behind the last token stay as they were
    return [y[: len(x)].cpu().numpy() for y in ys]


SHAPES = [  # tokens, inputs, outputs
    (1, 64, [1]), (1, 4096, [512, 33, 1]), (2, 128, [16]), (2, 1088, [100, 1]), (3, 576, [31, 32, 33]), (4, 1024, [130]), (5, 640, [17, 1, 1, 5]),
    (8, 4096, [96]), (9, 192, [40]), (17, 2048, [64, 64, 3]), (40, 1088, [257]), (1, 32768, [5]), (3, 24640, [18]), (11, 8192, [33]),
    (2, 512, [1, 2, 3, 4, 5, 6, 7, 8]),
    (64, 64, [1]), (65, 128, [129, 1]), (63, 4096, [520]), (100, 192, [128, 513]), (200, 512, [300, 64, 64]), (33, 4160, [40]), (20, 8192, [130]),
    (130, 1024, [1, 2, 600, 4, 5, 6, 7, 8]), (18, 12352, [33])]


@pytest.mark.parametrize("n,k,outs", SHAPES)
def test_products(pkg, n, k, outs):
    rng = np.random.default_rng(1000 + n * 7 + k)
    c = context(pkg, max_batch=256)
    mats = [moe_ref.weights(rng, o, k) for o in outs]
    x = rng.standard_normal((n, k)).astype(np.float32)
    for got, m in zip(run(pkg, c, mats, x), mats):
        moe_ref.close(got, *moe_ref.product(x, m))
    c.close()


LONG_SHAPES = [  # many tokens, rows enough that the weights are widened once for all of them
    (300, 64, [1300]), (513, 128, [400, 300, 1]), (301, 192, [1025]), (257, 576, [1281, 3]), (400, 1088, [900]), (320, 2112, [1000, 100]),
    (290, 4096, [1100]), (97, 4160, [2850]), (300, 8192, [1100]), (289, 8256, [1024, 1, 127]), (304, 12352, [960])]


@pytest.mark.parametrize("n,k,outs", LONG_SHAPES)
def test_products_of_many_tokens(pkg, n, k, outs):
    rng = np.random.default_rng(7000 + n * 7 + k)
    c = context(pkg, max_batch=1024)
    mats = [moe_ref.weights(rng, o, k) for o in outs]
    x = rng.standard_normal((n, k)).astype(np.float32)
    for got, m in zip(run(pkg, c, mats, x), mats):
        moe_ref.close(got, *moe_ref.product(x, m))
    c.close()


@pytest.mark.parametrize("k", [64, 192, 512, 1088, 4096, 4160])
@pytest.mark.parametrize("n,out", [(1, 130), (5, 130), (40, 130), (300, 1100)])
def test_scales_at_every_even_address(pkg, n, k, out):
    """Scales and biases need no more than their type's alignment, and what stands around them is not used."""
    rng = np.random.default_rng(n + k)
    c = context(pkg, max_batch=512)
    mat = moe_ref.weights(rng, out, k)
    x = rng.standard_normal((n, k)).astype(np.float32)
    want, bound = moe_ref.product(x, mat)
    xd, words = torch.from_numpy(x).cuda(), torch.from_numpy(mat[0].view(np.int32)).cuda()
    size = out * (k // 64)
    for s_at, b_at in [(0, 0), (1, 0), (2, 7), (5, 3), (4, 4), (7, 6)]:
        views = []
        for at, part in ((s_at, mat[1]), (b_at, mat[2])):
            block = torch.full((size + 32,), float("nan"), device="cuda", dtype=torch.bfloat16)
            views.append(block[8 + at: 8 + at + size].view(out, k // 64))
            views[-1].copy_(torch.from_numpy(part.view(np.int16)).cuda().view(torch.bfloat16).view(out, k // 64))
        y = torch.full((n, out), 7.0, device="cuda")
        c.proj_forward([pkg.proj_weights(words, *views)], n, xd, [y])
        c.synchronize()
        moe_ref.close(y.cpu().numpy(), want, bound)
    c.close()


@pytest.mark.parametrize("n", [1, 4, 13, 40])
def test_inputs_of_every_size(pkg, n):
    """Outliers beside small values, groups of zeros, values at both ends of fp32's range: no group loses its own."""
    rng = np.random.default_rng(5 + n)
    c = context(pkg)
    k = 64 * 12
    m = moe_ref.weights(rng, 48, k)
    x = rng.standard_normal((n, k))
    x[:, 64:128] = 0.0
    x[:, 128] = 3.0e4
    x[:, 192:256] *= 1e-6
    x[-1, :] = 0.0
    for scale in (1.0, 1e-30, 1e30):
        xs = (x * scale).astype(np.float32)
        want, bound = moe_ref.product(xs, m)
        moe_ref.close(run(pkg, c, [m], xs)[0], want, bound + 1e-300)
    c.close()


def test_non_finite_inputs_stay_in_their_token(pkg):
    rng = np.random.default_rng(3)
    for n in (4, 24):
        c = context(pkg)
        m = moe_ref.weights(rng, 40, 256)
        x = rng.standard_normal((n, 256)).astype(np.float32)
        want, bound = moe_ref.product(x, m)
        x[1, 3], x[3, 200] = np.inf, np.nan
        got = run(pkg, c, [m], x)[0]
        assert np.isnan(got[[1, 3]]).all()
        keep = [t for t in range(n) if t not in (1, 3)]
        moe_ref.close(got[keep], want[keep], bound[keep])
        c.close()


def test_host_pointers_and_uploaded_weights(pkg):
    rng = np.random.default_rng(8)
    c = context(pkg, host=True)
    mats = [moe_ref.weights(rng, o, 512) for o in (70, 9)]
    dev = [c.proj_upload(*m) for m in mats]
    for n in (1, 6, 64):
        x = rng.standard_normal((n, 512)).astype(np.float32)
        ys = [np.empty((n, 70), np.float32), np.empty((n, 9), np.float32)]
        c.proj_forward(dev, n, x, ys)
        for y, m in zip(ys, mats):
            moe_ref.close(y, *moe_ref.product(x, m))
    for d in dev:
        c.proj_free(d)
    c.close()


def test_same_token_gives_the_same_bits_wherever_it_stands(pkg):
    rng = np.random.default_rng(9)
    c = context(pkg)
    m = moe_ref.weights(rng, 65, 1024)
    x = rng.standard_normal((1, 1024)).astype(np.float32)
    for n in (2, 7, 8):
        got = run(pkg, c, [m], np.repeat(x, n, 0))[0]
        assert np.all(got == got[0])
    c.close()


@pytest.mark.parametrize("n", [1, 18])
def test_a_matrix_beyond_four_gigabytes(pkg, n):
    """Offsets past 32 bits: rows at both ends of a 4.4 GB matrix."""
    out, k = 270000, 32768
    gen = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randint(-2 ** 31, 2 ** 31, (out, k // 8), generator=gen, device="cuda", dtype=torch.int32)
    scales = (0.002 + 0.006 * torch.rand((out, k // 64), generator=gen, device="cuda")).bfloat16()
    biases = (-7.5 * scales.float()).bfloat16()
    x = torch.randn((n, k), generator=gen, device="cuda")
    y = torch.empty((n, out), device="cuda")
    c = context(pkg)
    c.proj_forward([pkg.proj_weights(w, scales, biases)], n, x, [y])
    c.synchronize()
    rows = torch.tensor([0, 1, 131071, 131072, 262143, 262144, out - 2, out - 1], device="cuda")
    m = (w[rows].cpu().numpy().view(np.uint32), scales[rows].view(torch.int16).cpu().numpy().view(np.uint16), biases[rows].view(torch.int16).cpu().numpy().view(np.uint16))
    moe_ref.close(y[:, rows].cpu().numpy(), *moe_ref.product(x.cpu().numpy(), m))
    c.close()


def test_two_contexts_at_once(pkg):
    """Contexts on streams of their own do not share anything: their calls may overlap."""
    rng = np.random.default_rng(77)
    m = moe_ref.weights(rng, 700, 1024)
    work = []
    for n in (3, 150):
        c = context(pkg, max_batch=256)
        st = torch.cuda.Stream()
        c.set_stream(st.cuda_stream)
        x = rng.standard_normal((n, 1024)).astype(np.float32)
        work.append((c, st, x, torch.from_numpy(x).cuda(), torch.empty((n, 700), device="cuda"), on_device(pkg, m)))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, st, x, xd, y, d in work:
            c.proj_forward([d], len(x), xd, [y])
    for c, st, x, xd, y, d in work:
        c.synchronize()
        moe_ref.close(y.cpu().numpy(), *moe_ref.product(x, m))
        c.close()


def test_more_rows_than_32_bit_row_numbers_take_are_refused(pkg):
    """The kernels count rows in int, past the last one by up to a unit."""
    c = context(pkg, max_batch=128)
    a = on_device(pkg, moe_ref.weights(np.random.default_rng(2), 16, 128))
    x, y = torch.zeros((100, 128), device="cuda"), torch.zeros((100, 16), device="cuda")
    for rows in (2 ** 30 + 1, 2 ** 31 - 1):
        big = pkg.binding.FmProjWeights.from_buffer_copy(a)
        big.out_dim = rows
        for n in (1, 100):
            with pytest.raises(pkg.FmError) as e:
                c.proj_forward([big], n, x, [y])
            assert e.value.status == pkg.binding.FM_ERR_UNSUPPORTED
    c.close()


def test_refusals(pkg):
    rng = np.random.default_rng(2)
    c = context(pkg, max_batch=8)
    a, b = on_device(pkg, moe_ref.weights(rng, 16, 128)), on_device(pkg, moe_ref.weights(rng, 16, 192))
    x, y = torch.zeros((9, 192), device="cuda"), torch.full((9, 16), 7.0, device="cuda")
    B = pkg.binding

    def status(ws, n, x_=x, ys=(y,)):
        with pytest.raises(pkg.FmError) as e:
            c.proj_forward(list(ws), n, x_, list(ys))
        assert e.value.text.startswith("fm_proj_forward")
        return e.value.status

    def changed(mat, **kw):
        r = B.FmProjWeights.from_buffer_copy(mat)
        for k, v in kw.items():
            setattr(r, k, v)
        return r
    assert status([a, b], 1, ys=(y, y)) == B.FM_ERR_INVALID                    # inputs of different length
    assert status([a], 9) == B.FM_ERR_INVALID and status([a], -1) == B.FM_ERR_INVALID
    assert status([a] * 9, 1, ys=[y] * 9) == B.FM_ERR_INVALID and status([], 1, ys=[]) == B.FM_ERR_INVALID
    assert status([a], 1, x_=None) == B.FM_ERR_INVALID and status([a], 1, ys=[None]) == B.FM_ERR_INVALID
    for bad in (dict(group_size=32), dict(in_dim=96), dict(in_dim=0), dict(out_dim=0), dict(format=1), dict(in_dim=65600)):
        assert status([changed(a, **bad)], 1) == B.FM_ERR_UNSUPPORTED
    assert status([changed(a, scales=None)], 1) == B.FM_ERR_INVALID
    assert status([changed(a, w=a.w + 4)], 1) == B.FM_ERR_INVALID
    assert status([a], 1, x_=x.view(-1)[1:129]) == B.FM_ERR_INVALID            # x off its 16-byte boundary
    assert status([changed(a, scales=a.scales + 1)], 1) == B.FM_ERR_INVALID and status([changed(a, biases=a.biases + 1)], 1) == B.FM_ERR_INVALID
    c.proj_forward([a], 0, x, [y])                                             # no tokens: nothing to do
    c.synchronize()
    assert torch.all(y == 7.0)
    c.close()
