"""fm_moe_experts against the chain in 64 bits, and the whole run router -> routing -> experts."""
import numpy as np
import pytest
import torch

import moe_ref
from test_gpu_proj_forward import context, on_device

pytestmark = pytest.mark.gpu


def stacks(rng, experts, hidden, inter):
    return (moe_ref.weights(rng, inter, hidden, (experts,)), moe_ref.weights(rng, inter, hidden, (experts,)), moe_ref.weights(rng, hidden, inter, (experts,)))


def cuda(a):
    if a is None:
        return None
    a = np.ascontiguousarray(a)
    if a.dtype == np.uint16:
        return torch.from_numpy(a.view(np.int16)).cuda().view(torch.bfloat16)
    return torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).cuda()


def device_stacks(pkg, m, first=0):
    return pkg.expert_weights(*(tuple(cuda(a) for a in s) for s in m), first_expert=first)


def inputs(rng, n, hidden, experts, top):
    x, res = rng.standard_normal((2, n, hidden)).astype(np.float32)
    ids = np.stack([rng.permutation(experts)[:top] for _ in range(n)]).astype(np.int32)
    w = rng.uniform(0.05, 0.5, size=(n, top)).astype(np.float32)
    return x, res, ids, w, moe_ref.bf16(1.0 + 0.1 * rng.standard_normal(hidden))


def run(pkg, c, dev, x, ids, w, res, nw, norm=True):
    n, hidden = x.shape
    out = torch.full((n + 1, hidden), 7.0, device="cuda")
    nrm = torch.full((n + 1, hidden), 7.0, device="cuda") if norm else None
    c.moe_experts(dev, n, ids.shape[1], cuda(x), cuda(ids), cuda(w), cuda(res), cuda(nw), out, nrm)
    c.synchronize()
    assert torch.all(out[n:] == 7.0) and (nrm is None or torch.all(nrm[n:] == 7.0))
    return out[:n].cpu().numpy(), None if nrm is None else nrm[:n].cpu().numpy()


def check(got, m, x, ids, w, res, nw, first=0):
    h, hn, bound = moe_ref.experts(*m, x, ids, w, res, nw, first)
    moe_ref.close(got[0], h, bound + 1e-300)
    if got[1] is not None:
        moe_ref.close(got[1], hn, moe_ref.norm_bound(h, bound, nw) + 1e-300)


SHAPES = [  # tokens, hidden, inter, experts, slots
    (1, 64, 64, 1, 1), (1, 256, 192, 8, 2), (1, 1024, 512, 16, 10), (3, 256, 192, 8, 2), (2, 128, 64, 5, 3), (5, 192, 320, 4, 4), (9, 576, 128, 40, 6),
    (30, 128, 192, 6, 2), (64, 256, 64, 3, 1), (70, 128, 128, 100, 8), (33, 1088, 704, 5, 3), (150, 192, 128, 2, 2), (7, 64, 64, 40, 32),
    (260, 512, 320, 4, 2), (400, 256, 512, 3, 1)]


@pytest.mark.parametrize("n,hidden,inter,experts,top", SHAPES)
def test_against_64_bits(pkg, n, hidden, inter, experts, top):
    rng = np.random.default_rng(n * 31 + hidden + experts)
    c = context(pkg, max_batch=512)
    m = stacks(rng, experts, hidden, inter)
    x, res, ids, w, nw = inputs(rng, n, hidden, experts, top)
    check(run(pkg, c, device_stacks(pkg, m), x, ids, w, res, nw), m, x, ids, w, res, nw)
    check(run(pkg, c, device_stacks(pkg, m), x, ids, w, None, None, norm=False), m, x, ids, w, None, None)
    c.close()


@pytest.mark.parametrize("n", [1, 4, 41, 130])
def test_slots_without_an_expert_here(pkg, n):
    """Other ranks' experts, -1, ids beyond all experts; tokens with no expert here keep their residual; one id twice."""
    rng = np.random.default_rng(n)
    c = context(pkg, max_batch=256)
    m = stacks(rng, 5, 128, 192)
    x, res, ids, w, nw = inputs(rng, n, 128, 16, 4)
    ids[0] = [-1, 3, 2 ** 30, -2 ** 31]
    if n > 2:
        ids[1] = [7, 7, 7, -1]
    for first in (0, 4, 11):
        got = run(pkg, c, device_stacks(pkg, m, first), x, ids, w, res, nw)
        check(got, m, x, ids, w, res, nw, first)
        if first == 4:
            assert np.array_equal(got[0][0], res[0])
    c.close()


def test_everything_to_one_expert(pkg):
    rng = np.random.default_rng(12)
    c = context(pkg, max_batch=256)
    m = stacks(rng, 9, 192, 64)
    x, res, ids, w, nw = inputs(rng, 200, 192, 9, 2)
    ids[:] = [8, 3]
    check(run(pkg, c, device_stacks(pkg, m), x, ids, w, res, nw), m, x, ids, w, res, nw)
    c.close()


@pytest.mark.parametrize("n", [1, 20, 140])
def test_one_blob_per_expert(pkg, n):
    """All nine arrays of an expert in one block, a fixed distance apart."""
    rng = np.random.default_rng(21 + n)
    c = context(pkg, max_batch=256)
    E, hidden, inter = 6, 192, 128
    m = stacks(rng, E, hidden, inter)
    flat = [a for s in m for a in s]
    sizes = [a[0].nbytes for a in flat]
    at = np.cumsum([0] + [(s + 15) // 16 * 16 for s in sizes])
    stride = int(at[-1]) + 48
    blob = np.zeros((E, stride), np.uint8)
    for a, o, s in zip(flat, at, sizes):
        blob[:, o:o + s] = a.reshape(E, -1).view(np.uint8)
    d = torch.from_numpy(blob).cuda()
    dev = pkg.binding.FmExpertWeights(0, E, 0, hidden, inter, 64, stride, *(d.data_ptr() + int(o) for o in at[:-1]))
    x, res, ids, w, nw = inputs(rng, n, hidden, E, 3)
    check(run(pkg, c, dev, x, ids, w, res, nw), m, x, ids, w, res, nw)
    c.close()


@pytest.mark.parametrize("n", [2, 100])
def test_experts_beyond_four_gigabytes(pkg, n):
    """One blob per expert, 64 MB apart: the last of 80 lies 5 GB behind the first."""
    rng = np.random.default_rng(90 + n)
    c = context(pkg, max_batch=128)
    E, hidden, inter, stride = 80, 128, 64, 64 << 20
    few = [0, 31, 63, 64, 79]
    m = stacks(rng, len(few), hidden, inter)
    blob = torch.empty(E * stride, dtype=torch.uint8, device="cuda")
    at, o = [], 0
    for a in (a for s in m for a in s):
        at.append(o)
        flat = np.ascontiguousarray(a.reshape(len(few), -1)).view(np.uint8)
        for i, e in enumerate(few):
            blob[e * stride + o: e * stride + o + flat.shape[1]] = torch.from_numpy(flat[i]).cuda()
        o += (flat.shape[1] + 15) // 16 * 16
    dev = pkg.binding.FmExpertWeights(0, E, 0, hidden, inter, 64, stride, *(blob.data_ptr() + a for a in at))
    x, res, ids, w, nw = inputs(rng, n, hidden, len(few), 3)
    got = run(pkg, c, dev, x, np.array(few, np.int32)[ids], w, res, nw)
    check(got, m, x, ids, w, res, nw)
    c.close()


def test_in_place_and_host_pointers(pkg):
    rng = np.random.default_rng(30)
    m = stacks(rng, 7, 128, 64)
    c = context(pkg, max_batch=64)
    dev = device_stacks(pkg, m)
    for n in (1, 50):
        x, res, ids, w, nw = inputs(rng, n, 128, 7, 3)
        h, nrm = cuda(res), cuda(x)
        c.moe_experts(dev, n, 3, nrm, cuda(ids), cuda(w), h, cuda(nw), h, nrm)  # h_out over the residual, h_norm over x
        c.synchronize()
        check((h.cpu().numpy(), nrm.cpu().numpy()), m, x, ids, w, res, nw)
        c.set_pointer_mode(pkg.binding.FM_PTR_HOST)
        out, nrm = np.empty_like(x), np.empty_like(x)
        c.moe_experts(dev, n, 3, x, ids, w, res, nw, out, nrm)
        check((out, nrm), m, x, ids, w, res, nw)
        c.set_pointer_mode(pkg.binding.FM_PTR_DEVICE)
    c.close()


def test_the_same_call_gives_the_same_bits(pkg):
    rng = np.random.default_rng(31)
    c = context(pkg, max_batch=256)
    m = stacks(rng, 11, 256, 128)
    dev = device_stacks(pkg, m)
    for n in (1, 30, 200):
        x, res, ids, w, nw = inputs(rng, n, 256, 11, 4)
        a = run(pkg, c, dev, x, ids, w, res, nw)
        for _ in range(3):
            b = run(pkg, c, dev, x, ids, w, res, nw)
            assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    c.close()


def test_router_routing_and_experts_as_one_run(pkg):
    """The end of a layer as a host runs it -- router logits with the shared expert's gate, routing, experts with the shared
    one stacked behind them, the next layer's projections -- eagerly, on another stream, and as a captured graph replayed."""
    rng = np.random.default_rng(40)
    E, hidden, inter, top = 12, 256, 128, 3
    c = context(pkg, max_batch=256)
    m = stacks(rng, E + 1, hidden, inter)
    router, nxt = moe_ref.weights(rng, E + 1, hidden), moe_ref.weights(rng, 96, hidden)
    router = (router[0], moe_ref.bf16(4 * moe_ref.f32(router[1])), moe_ref.bf16(4 * moe_ref.f32(router[2])))
    dev, d_router, d_next = device_stacks(pkg, m), on_device(pkg, router), on_device(pkg, nxt)
    rcd = dict(num_experts=E, top_k=top, score=0, num_groups=1, top_groups=1, group_best=1, renormalize=1, scale=1.0, shared_expert=1)
    rc = pkg.route_config(**rcd)
    for n in (1, 6, 180):
        bufs = dict(logits=torch.empty((n, E + 1), device="cuda"), ids=torch.empty((n, top + 1), device="cuda", dtype=torch.int32),
                    w=torch.empty((n, top + 1), device="cuda"), h=torch.empty((n, hidden), device="cuda"), hn=torch.empty((n, hidden), device="cuda"),
                    y=torch.empty((n, 96), device="cuda"), x=torch.empty((n, hidden), device="cuda"), res=torch.empty((n, hidden), device="cuda"))
        nw = moe_ref.bf16(1.0 + 0.1 * rng.standard_normal(hidden))
        d_nw = cuda(nw)

        def chain():
            c.proj_forward([d_router], n, bufs["x"], [bufs["logits"]])
            c.moe_route(rc, n, bufs["logits"], None, bufs["ids"], bufs["w"])
            c.moe_experts(dev, n, top + 1, bufs["x"], bufs["ids"], bufs["w"], bufs["res"], d_nw, bufs["h"], bufs["hn"])
            c.proj_forward([d_next], n, bufs["hn"], [bufs["y"]])

        def verify(x, res):
            logits = bufs["logits"].cpu().numpy()
            moe_ref.close(logits, *moe_ref.product(x, router))
            ids, w = moe_ref.route(logits, None, rcd)
            assert np.array_equal(bufs["ids"].cpu().numpy(), ids)
            got_w = bufs["w"].cpu().numpy()
            assert np.all(np.abs(got_w - w) <= 128 * moe_ref.EPS * w)
            check((bufs["h"].cpu().numpy(), bufs["hn"].cpu().numpy()), m, x, ids, got_w, res, nw)
            moe_ref.close(bufs["y"].cpu().numpy(), *moe_ref.product(bufs["hn"].cpu().numpy(), nxt))

        def load():
            x, res = rng.standard_normal((2, n, hidden)).astype(np.float32)
            bufs["x"].copy_(torch.from_numpy(x)); bufs["res"].copy_(torch.from_numpy(res))
            for k in ("logits", "ids", "w", "h", "hn", "y"):
                bufs[k].fill_(-1)
            return x, res

        x, res = load()
        chain(); c.synchronize()
        verify(x, res)
        side = torch.cuda.Stream()
        x, res = load()
        side.wait_stream(torch.cuda.current_stream())
        c.set_stream(side.cuda_stream)
        chain(); c.synchronize()
        verify(x, res)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.set_stream(torch.cuda.current_stream().cuda_stream)
            chain()
        c.set_stream(torch.cuda.current_stream().cuda_stream)
        for _ in range(2):
            x, res = load()
            g.replay()
            torch.cuda.synchronize()
            verify(x, res)
        del g
    c.close()


def test_growing_the_workspace_keeps_captured_graphs_valid(pkg):
    rng = np.random.default_rng(50)
    c = context(pkg, max_batch=256)
    m = stacks(rng, 5, 128, 64)
    dev = device_stacks(pkg, m)
    x, res, ids, w, nw = inputs(rng, 4, 128, 5, 2)
    d = [cuda(a) for a in (x, ids, w, res, nw)]
    out, nrm = torch.empty((4, 128), device="cuda"), torch.empty((4, 128), device="cuda")
    call = lambda: c.moe_experts(dev, 4, 2, d[0], d[1], d[2], d[3], d[4], out, nrm)  # noqa: E731
    g = torch.cuda.CUDAGraph()
    with pytest.raises(pkg.FmError) as e:  # the first call of a size allocates: refused inside a capture
        with torch.cuda.graph(g):
            c.set_stream(torch.cuda.current_stream().cuda_stream)
            call()
    assert e.value.status == pkg.binding.FM_ERR_CAPACITY
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.set_stream(torch.cuda.current_stream().cuda_stream)
        call()
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    x2, res2, ids2, w2, nw2 = inputs(rng, 250, 128, 5, 3)
    run(pkg, c, dev, x2, ids2, w2, res2, nw2)  # a larger call moves the workspace
    out.fill_(-1); nrm.fill_(-1)
    g.replay()
    torch.cuda.synchronize()
    check((out.cpu().numpy(), nrm.cpu().numpy()), m, x, ids, w, res, nw)
    del g
    c.close()


def test_refusals(pkg):
    rng = np.random.default_rng(60)
    c = context(pkg, max_batch=8)
    dev = device_stacks(pkg, stacks(rng, 3, 128, 64))
    x = torch.zeros((9, 128), device="cuda")
    ids, w = torch.zeros((9, 2), device="cuda", dtype=torch.int32), torch.zeros((9, 2), device="cuda")
    out = torch.full((9, 128), 7.0, device="cuda")
    B = pkg.binding

    def status(n=1, top=2, x_=x, ids_=ids, w_=w, res=None, out_=out, nrm=None, **kw):
        d = B.FmExpertWeights.from_buffer_copy(dev)
        for k, v in kw.items():
            setattr(d, k, v)
        with pytest.raises(pkg.FmError) as e:
            c.moe_experts(d, n, top, x_, ids_, w_, res, None, out_, nrm)
        assert e.value.text.startswith("fm_moe_experts")
        return e.value.status
    for bad in (dict(format=1), dict(group_size=128), dict(hidden=96), dict(inter=0), dict(inter=65600), dict(num_experts=0), dict(num_experts=1025), dict(top=0), dict(top=33)):
        assert status(**bad) == B.FM_ERR_UNSUPPORTED
    for bad in (dict(first_expert=-1), dict(expert_stride=-16), dict(expert_stride=24), dict(n=9), dict(n=-1), dict(gate_w=None), dict(down_biases=None), dict(up_w=dev.up_w + 8), dict(down_scales=dev.down_scales + 1),
                dict(x_=None), dict(ids_=None), dict(w_=None), dict(out_=None), dict(x_=x.view(-1)[1:129]), dict(out_=out.view(-1)[1:129]), dict(nrm=out.view(-1)[2:130]),
                dict(res=x.view(-1)[3:131])):
        assert status(**bad) == B.FM_ERR_INVALID
    assert status(total_experts=-1) == status(total_experts=2) == status(total_experts=5, first_expert=3) == B.FM_ERR_INVALID
    c.moe_experts(dev, 0, 2, x, ids, w, None, None, out, None)
    c.synchronize()
    assert torch.all(out == 7.0)
    c.close()
