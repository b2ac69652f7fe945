"""fm_proj_forward and fm_moe_experts choose among kernels by size: each choice, at the places where it can go wrong."""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import moe_ref
from test_gpu_moe_experts import check, cuda, device_stacks, inputs, run as run_experts, stacks
from test_gpu_proj_forward import context, on_device, run as run_proj

pytestmark = pytest.mark.gpu

PROJ = [(1, 5, 768, 48), (1, 40, 768, 48), (2, 300, 768, 1000)]  # launches, tokens, inputs, outputs
EXPERTS = [(3, 6, 192, 128), (4, 300, 192, 128), (6, 700, 512, 320)]  # launches, tokens, hidden, inter (5 or 6 experts, 3 slots)


def launches(c, call):
    before = c.launch_count()
    result = call()
    return c.launch_count() - before, result


@pytest.mark.parametrize("many,n,k,out", PROJ)
def test_projection_inputs_of_every_size(pkg, many, n, k, out):
    """Outliers beside small values, groups of zeros, values at both ends of fp32's range; infinities and NaN stay in their token."""
    rng = np.random.default_rng(500 + n)
    c = context(pkg, max_batch=512)
    m = moe_ref.weights(rng, out, k)
    x = rng.standard_normal((n, k))
    x[:, 64:128] = 0.0
    x[:, 128] = 3.0e4
    x[:, 192:256] *= 1e-6
    x[-1, :] = 0.0
    for scale in (1.0, 1e-30, 1e30):
        xs = (x * scale).astype(np.float32)
        want, bound = moe_ref.product(xs, m)
        count, got = launches(c, lambda: run_proj(pkg, c, [m], xs)[0])
        assert count == many
        moe_ref.close(got, want, bound + 1e-300)
    xs = x.astype(np.float32)
    want, bound = moe_ref.product(xs, m)
    xs[1, 3], xs[3, 200] = np.inf, np.nan
    got = run_proj(pkg, c, [m], xs)[0]
    assert np.isnan(got[[1, 3]]).all()
    keep = [t for t in range(n) if t not in (1, 3)]
    moe_ref.close(got[keep], want[keep], bound[keep])
    c.close()


WIDE_AND_NOT = [(1, 8, 1024, 48), (1, 40, 1024, 48), (2, 300, 1024, 1000), (2, 300, 832, 1000)]  # launches, tokens, inputs, outputs
RATIOS = [1e-2, 1e-3, 1e-4, 2.0 ** -7, 2.0 ** -8, 2.0 ** -12, 2.0 ** -16, 2.0 ** -20]


@pytest.mark.parametrize("ratio", RATIOS)
@pytest.mark.parametrize("many,n,k,out", WIDE_AND_NOT)
def test_groups_whose_scales_lie_far_apart(pkg, many, n, k, out, ratio):
    """Every group keeps its weights, however small its scale is beside its neighbours': with inputs of one size, with none but
    in the groups of small scales, and with inputs that make up for the scales."""
    rng = np.random.default_rng(620 + n + k)
    c = context(pkg, max_batch=512)
    m = moe_ref.spread(rng, moe_ref.weights(rng, out, k), ratio)
    big = np.repeat(np.arange(k // 64) % 4 == 1, 64)
    x = rng.standard_normal((n, k)).astype(np.float32)
    for xs in (x, np.where(big, 0, x), np.where(big, x * 64 * ratio, x)):
        xs = xs.astype(np.float32)
        count, got = launches(c, lambda: run_proj(pkg, c, [m], xs)[0])
        assert count == many
        moe_ref.close(got, *moe_ref.product(xs, m))
    c.close()


@pytest.mark.parametrize("ratio", [2.0 ** -20, 2.0 ** -24, 2.0 ** -28])
@pytest.mark.parametrize("many,n,k,out", [(1, 8, 4096, 48), (2, 300, 4096, 1000), (2, 300, 4160, 1000)])
def test_rows_whose_biases_lie_far_apart(pkg, many, n, k, out, ratio):
    """Every other 256 inputs have small scales and biases, and only those have inputs, all of one sign: the biases' share is
    what it takes the share of the nibbles to cancel."""
    rng = np.random.default_rng(660 + n + k)
    c = context(pkg, max_batch=512)
    w, s, b = moe_ref.weights(rng, out, k)
    small = np.arange(k // 64) // 4 % 2 == 1
    m = (w, *(moe_ref.bf16(np.where(small, moe_ref.f32(a) * ratio, moe_ref.f32(a))) for a in (s, b)))
    x = np.where(np.repeat(small, 64), np.abs(rng.standard_normal((n, k))), 0).astype(np.float32)
    count, got = launches(c, lambda: run_proj(pkg, c, [m], x)[0])
    assert count == many
    moe_ref.close(got, *moe_ref.product(x, m))
    c.close()


@pytest.mark.parametrize("ratio", [2.0 ** -12, 2.0 ** -16, 2.0 ** -20, 2.0 ** -22])
@pytest.mark.parametrize("many,n,k,out", WIDE_AND_NOT)
def test_small_inputs_beside_large_ones_without_weight(pkg, many, n, k, out, ratio):
    """Inputs that lie `ratio` below their token's largest, where the large ones meet weights of zero."""
    rng = np.random.default_rng(680 + n + k)
    c = context(pkg, max_batch=512)
    w, s, b = moe_ref.weights(rng, out, k)
    large = np.arange(k // 64) % 4 == 2
    m = (w, np.where(large, 0, s).astype(np.uint16), np.where(large, 0, b).astype(np.uint16))
    x = (rng.standard_normal((n, k)) * np.where(np.repeat(large, 64), 1, ratio)).astype(np.float32)
    count, got = launches(c, lambda: run_proj(pkg, c, [m], x)[0])
    assert count == many
    moe_ref.close(got, *moe_ref.product(x, m))
    c.close()


@pytest.mark.parametrize("many,n,k,out", [(1, 1, 768, 48), (1, 2, 832, 48), (1, 4, 768, 48), *PROJ])
def test_inputs_next_to_the_largest_number(pkg, many, n, k, out):
    """Finite inputs whose sums leave fp32's range do not make outputs that lie within it infinite or NaN."""
    rng = np.random.default_rng(700 + n)
    c = context(pkg, max_batch=512)
    w, s, b = moe_ref.weights(rng, out, k)
    m = (w, *(moe_ref.bf16(moe_ref.f32(a) / 128) for a in (s, b)))
    x = rng.uniform(2.0e38, 3.4e38, size=(n, k)).astype(np.float32)
    x[0, : k // 2] *= -1
    x[-1, ::3] = np.finfo(np.float32).max
    want, bound = moe_ref.product(x, m)
    assert np.abs(want).max() < 1e38
    count, got = launches(c, lambda: run_proj(pkg, c, [m], x)[0])
    assert count == many
    moe_ref.close(got, want, bound)
    c.close()


@pytest.mark.parametrize("ratio", [1e-3, 2.0 ** -20])
@pytest.mark.parametrize("many,n,hidden,inter", EXPERTS)
def test_experts_whose_scales_lie_far_apart(pkg, many, n, hidden, inter, ratio):
    rng = np.random.default_rng(640 + n)
    c = context(pkg, max_batch=1024)
    m = [moe_ref.spread(rng, a, ratio) for a in stacks(rng, 6, hidden, inter)]
    x, res, ids, w, nw = inputs(rng, n, hidden, 6, 3)
    x[:, np.repeat(np.arange(hidden // 64) % 4 == 1, 64)] = 0.0
    x /= np.float32(ratio)  # gate and up come out as large as usual
    count, got = launches(c, lambda: run_experts(pkg, c, device_stacks(pkg, m), x, ids, w, None, nw))
    assert count == many
    check(got, m, x, ids, w, None, nw)
    c.close()


@pytest.mark.parametrize("many,n,k,out", PROJ)
def test_projection_host_pointers_and_bits(pkg, many, n, k, out):
    """Host pointers give the bits that device pointers give, and equal tokens of a call equal rows."""
    rng = np.random.default_rng(510 + n)
    c = context(pkg, max_batch=512)
    m = moe_ref.weights(rng, out, k)
    d = on_device(pkg, m)
    x = rng.standard_normal((n, k)).astype(np.float32)
    x[n // 2] = x[0]
    got = run_proj(pkg, c, [m], x)[0]
    moe_ref.close(got, *moe_ref.product(x, m))
    assert np.array_equal(got[0], got[n // 2])
    c.set_pointer_mode(pkg.binding.FM_PTR_HOST)
    y = np.empty((n, out), np.float32)
    count, _ = launches(c, lambda: c.proj_forward([d], n, x, [y]))
    assert count == many and np.array_equal(y, got)
    c.close()


@pytest.mark.parametrize("n", [1, 8])
def test_a_few_tokens_are_captured_without_a_call_before(pkg, n):
    """Up to 8 tokens nothing is allocated, however many rows there are."""
    rng = np.random.default_rng(515 + n)
    c = context(pkg)
    m = moe_ref.weights(rng, 40000, 128)
    d = on_device(pkg, m)
    x, y = torch.zeros((n, 128), device="cuda"), torch.empty((n, 40000), device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.set_stream(torch.cuda.current_stream().cuda_stream)
        c.proj_forward([d], n, x, [y])
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    values = rng.standard_normal((n, 128)).astype(np.float32)
    x.copy_(torch.from_numpy(values))
    g.replay()
    torch.cuda.synchronize()
    moe_ref.close(y.cpu().numpy(), *moe_ref.product(values, m))
    del g
    c.close()


def test_projections_of_two_contexts_at_once(pkg):
    rng = np.random.default_rng(520)
    work = []
    for many, n, k, out in PROJ:
        m = moe_ref.weights(rng, out, k)
        c = context(pkg, max_batch=512)
        c.set_stream(torch.cuda.Stream().cuda_stream)
        x = rng.standard_normal((n, k)).astype(np.float32)
        work.append((c, x, cuda(x), torch.empty((n, out), device="cuda"), on_device(pkg, m), m))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, x, xd, y, d, m in work:
            c.proj_forward([d], len(x), xd, [y])
    for c, x, xd, y, d, m in work:
        c.synchronize()
        moe_ref.close(y.cpu().numpy(), *moe_ref.product(x, m))
        c.close()


def test_many_tokens_through_a_matrix_beyond_four_gigabytes(pkg):
    """Offsets past 32 bits where the weights are widened once for many tokens: rows at both ends of a 4.4 GB matrix."""
    out, k, n = 270000, 32768, 70
    gen = torch.Generator(device="cuda").manual_seed(2)
    w = torch.randint(-2 ** 31, 2 ** 31, (out, k // 8), generator=gen, device="cuda", dtype=torch.int32)
    scales = (0.002 + 0.006 * torch.rand((out, k // 64), generator=gen, device="cuda")).bfloat16()
    biases = (-7.5 * scales.float()).bfloat16()
    x, y = torch.randn((n, k), generator=gen, device="cuda"), torch.empty((n, out), device="cuda")
    c = context(pkg, max_batch=128)
    count, _ = launches(c, lambda: c.proj_forward([pkg.proj_weights(w, scales, biases)], n, x, [y]))
    c.synchronize()
    assert count == 2
    rows = torch.tensor([0, 131071, 131072, 262143, 262144, out - 1], device="cuda")
    m = (w[rows].cpu().numpy().view(np.uint32), scales[rows].view(torch.int16).cpu().numpy().view(np.uint16), biases[rows].view(torch.int16).cpu().numpy().view(np.uint16))
    moe_ref.close(y[:, rows].cpu().numpy(), *moe_ref.product(x.cpu().numpy(), m))
    c.close()


@pytest.mark.parametrize("many,n,hidden,inter", EXPERTS)
def test_slots_without_an_expert_here(pkg, many, n, hidden, inter):
    """Other ranks' experts, -1, ids beyond all experts, one id twice, a token without an expert here."""
    rng = np.random.default_rng(530 + n)
    c = context(pkg, max_batch=1024)
    m = stacks(rng, 5, hidden, inter)
    x, res, ids, w, nw = inputs(rng, n, hidden, 8, 3)
    ids[0] = [-1, 2 ** 30, -2 ** 31]
    ids[1], ids[2] = [6, 6, -1], [7, 6, 7]
    for first in (0, 3):
        count, got = launches(c, lambda: run_experts(pkg, c, device_stacks(pkg, m, first), x, ids, w, res, nw))
        assert count == many
        check(got, m, x, ids, w, res, nw, first)
        assert np.array_equal(got[0][0], res[0])
    c.close()


@pytest.mark.parametrize("many,n,hidden,inter", EXPERTS)
def test_everything_to_one_expert_or_to_none(pkg, many, n, hidden, inter):
    rng = np.random.default_rng(540 + n)
    c = context(pkg, max_batch=1024)
    m = stacks(rng, 6, hidden, inter)
    x, res, ids, w, nw = inputs(rng, n, hidden, 6, 3)
    ids[:] = [4, 4, -1]
    count, got = launches(c, lambda: run_experts(pkg, c, device_stacks(pkg, m), x, ids, w, res, nw))
    assert count == many
    check(got, m, x, ids, w, res, nw)
    ids[:] = -1
    got = run_experts(pkg, c, device_stacks(pkg, m), x, ids, w, res, nw)
    assert np.array_equal(got[0], res)
    c.close()


@pytest.mark.parametrize("many,n,hidden,inter", EXPERTS)
def test_non_finite_inputs_stay_in_their_token(pkg, many, n, hidden, inter):
    rng = np.random.default_rng(550 + n)
    c = context(pkg, max_batch=1024)
    m = stacks(rng, 6, hidden, inter)
    x, res, ids, w, nw = inputs(rng, n, hidden, 6, 3)
    h, hn, bound = moe_ref.experts(*m, x, ids, w, res, nw)
    x[1, 5], x[4, hidden - 1] = np.nan, -np.inf
    got = run_experts(pkg, c, device_stacks(pkg, m), x, ids, w, res, nw)
    assert np.isnan(got[0][1]).all() and np.isnan(got[0][4]).all()
    keep = [t for t in range(n) if t not in (1, 4)]
    moe_ref.close(got[0][keep], h[keep], bound[keep] + 1e-300)
    c.close()


@pytest.mark.parametrize("at", [0, 2, 6])
@pytest.mark.parametrize("many,n,hidden,inter", EXPERTS)
def test_one_blob_per_expert_and_scales_at_even_addresses(pkg, many, n, hidden, inter, at):
    rng = np.random.default_rng(560 + n)
    c = context(pkg, max_batch=1024)
    E = 5
    m = stacks(rng, E, hidden, inter)
    flat = [a for s in m for a in s]
    places, end = [], 0
    for a in flat:
        places.append(end + (at if a.dtype == np.uint16 else 0))
        end = (places[-1] + a[0].nbytes + 15) // 16 * 16
    blob = np.full((E, end + 32), 0xFF, np.uint8)  # NaN as bf16
    for a, o in zip(flat, places):
        blob[:, o:o + a[0].nbytes] = a.reshape(E, -1).view(np.uint8)
    d = torch.from_numpy(blob).cuda()
    dev = pkg.binding.FmExpertWeights(0, E, 0, hidden, inter, 64, end + 32, *(d.data_ptr() + o for o in places))
    x, res, ids, w, nw = inputs(rng, n, hidden, E, 3)
    count, got = launches(c, lambda: run_experts(pkg, c, dev, x, ids, w, res, nw))
    assert count == many
    check(got, m, x, ids, w, res, nw)
    c.close()


@pytest.mark.parametrize("many,n", [(3, 2), (4, 100), (6, 1100)])
def test_experts_beyond_four_gigabytes(pkg, many, n):
    """One blob per expert, 64 MB apart: the last of 80 lies 5 GB behind the first."""
    rng = np.random.default_rng(570 + n)
    c = context(pkg, max_batch=2048)
    E, hidden, inter, stride = 80, 512, 320, 64 << 20
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
    count, got = launches(c, lambda: run_experts(pkg, c, dev, x, np.array(few, np.int32)[ids], w, res, nw))
    assert count == many
    check(got, m, x, ids, w, res, nw)
    c.close()


@pytest.mark.parametrize("many,n,hidden,inter", EXPERTS)
def test_in_place_host_pointers_and_replay(pkg, many, n, hidden, inter):
    """h_out over the residual and h_norm over x; host pointers; a captured call replayed with new inputs: the same bits."""
    rng = np.random.default_rng(580 + n)
    c = context(pkg, max_batch=1024)
    m = stacks(rng, 6, hidden, inter)
    dev = device_stacks(pkg, m)
    x, res, ids, w, nw = inputs(rng, n, hidden, 6, 3)
    want = run_experts(pkg, c, dev, x, ids, w, res, nw)
    check(want, m, x, ids, w, res, nw)
    d = [cuda(a) for a in (x, ids, w, res, nw)]
    c.moe_experts(dev, n, 3, d[0], d[1], d[2], d[3], d[4], d[3], d[0])
    c.synchronize()
    assert np.array_equal(d[3].cpu().numpy(), want[0]) and np.array_equal(d[0].cpu().numpy(), want[1])
    c.set_pointer_mode(pkg.binding.FM_PTR_HOST)
    out, nrm = np.empty_like(x), np.empty_like(x)
    c.moe_experts(dev, n, 3, x, ids, w, res, nw, out, nrm)
    assert np.array_equal(out, want[0]) and np.array_equal(nrm, want[1])
    c.set_pointer_mode(pkg.binding.FM_PTR_DEVICE)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.set_stream(torch.cuda.current_stream().cuda_stream)
        c.moe_experts(dev, n, 3, d[0], d[1], d[2], d[3], d[4], d[3], d[0])
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        x, res, ids, w, _ = inputs(rng, n, hidden, 6, 3)
        want = run_experts(pkg, c, dev, x, ids, w, res, nw)
        for to, a in zip(d, (x, ids, w, res)):
            to.copy_(torch.from_numpy(a))
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(d[3].cpu().numpy(), want[0]) and np.array_equal(d[0].cpu().numpy(), want[1])
    del g
    c.close()


def test_total_experts_changes_the_choice_and_not_the_answer(pkg):
    rng = np.random.default_rng(590)
    c = context(pkg, max_batch=1024)
    m = stacks(rng, 6, 512, 320)
    x, res, ids, w, nw = inputs(rng, 700, 512, 48, 3)
    counts = []
    for total in (0, 48):
        dev = device_stacks(pkg, m)
        dev.total_experts = total
        count, got = launches(c, lambda: run_experts(pkg, c, dev, x, ids, w, res, nw))
        check(got, m, x, ids, w, res, nw)
        counts.append(count)
    assert counts == [6, 4]
    c.close()


@pytest.mark.parametrize("many,n,out", [(1, 1, 33), (1, 8, 33), (1, 17, 33), (2, 600, 330)])
def test_projection_of_the_longest_input(pkg, many, n, out):
    rng = np.random.default_rng(600 + n)
    c = context(pkg, max_batch=1024)
    m = moe_ref.weights(rng, out, 65536)
    x = rng.standard_normal((n, 65536)).astype(np.float32)
    count, got = launches(c, lambda: run_proj(pkg, c, [m], x)[0])
    assert count == many
    moe_ref.close(got, *moe_ref.product(x, m))
    c.close()


@pytest.mark.parametrize("n,hidden,inter", [(2, 65536, 64), (2, 64, 65536), (40, 65536, 64), (40, 64, 65536), (900, 8192, 64), (900, 64, 8192)])
def test_experts_of_the_longest_rows(pkg, n, hidden, inter):
    rng = np.random.default_rng(610 + n)
    c = context(pkg, max_batch=1024)
    m = stacks(rng, 2, hidden, inter)
    x, res, ids, w, nw = inputs(rng, n, hidden, 2, 2)
    check(run_experts(pkg, c, device_stacks(pkg, m), x, ids, w, res, nw), m, x, ids, w, res, nw)
    c.close()


def test_host_pointers_of_a_context_with_few_heads(pkg):
    """A context stages as many tokens as it was made for, however small its attention tensors are."""
    rng = np.random.default_rng(720)
    n, hidden = 512, 2048
    few = dict(num_attn_heads=4, num_kv_heads=1, linear_num_v_heads=1, linear_num_k_heads=1)
    c = context(pkg, host=True, max_batch=n, **few)
    m, mat = stacks(rng, 3, hidden, 64), moe_ref.weights(rng, 9000, 128)
    dev, d = device_stacks(pkg, m), on_device(pkg, mat)
    rcd = dict(num_experts=1024, top_k=30, score=1, num_groups=1, top_groups=1, group_best=1, renormalize=1, scale=1.0, shared_expert=1)

    def project():
        x, y = rng.standard_normal((n, 128)).astype(np.float32), np.empty((n, 9000), np.float32)
        c.proj_forward([d], n, x, [y])
        moe_ref.close(y, *moe_ref.product(x, mat))

    def route():
        logits = rng.standard_normal((n, 1025)).astype(np.float32)
        ids, w = np.empty((n, 31), np.int32), np.empty((n, 31), np.float32)
        c.moe_route(pkg.route_config(**rcd), n, logits, None, ids, w)
        want = moe_ref.route(logits, None, rcd)
        assert np.array_equal(ids, want[0]) and np.abs(w - want[1]).max() < 1e-6

    def experts():
        x, res, ids, w, nw = inputs(rng, n, hidden, 3, 2)
        out, nrm = np.empty_like(x), np.empty_like(x)
        c.moe_experts(dev, n, 2, x, ids, w, res, nw, out, nrm)
        check((out, nrm), m, x, ids, w, res, nw)
    route()
    experts()
    project()
    experts()
    route()
    c.close()
    c = context(pkg, host=True, max_batch=n, **few)
    project()
    c.close()


THREADS = """
import sys, threading
sys.path[:0] = {path!r}
import numpy as np, torch
import moe_ref
from __graft_entry__ import load_package
from test_gpu_moe_experts import check, cuda, device_stacks, inputs, stacks
from test_gpu_proj_forward import context, on_device
pkg = load_package()
rng = np.random.default_rng(730)
mat, m = moe_ref.weights(rng, 1100, 512), stacks(rng, 6, 512, 320)
d, dev = on_device(pkg, mat), device_stacks(pkg, m)
sizes = [1, 2, 4, 8, 300, 700]
work = [(n, inputs(rng, n, 512, 6, 3)) for n in sizes]
contexts = [context(pkg, max_batch=1024) for _ in range(4)]
buffers = [[([cuda(a) for a in v], torch.empty((n, 1100), device="cuda"), torch.empty((n, 512), device="cuda"), torch.empty((n, 512), device="cuda")) for n, v in work]
           for _ in contexts]
streams = [torch.cuda.Stream() for _ in contexts]
torch.cuda.synchronize()
gate, failed = threading.Barrier(len(contexts)), []

def body(c, st, bufs):
    try:
        c.set_stream(st.cuda_stream)
        gate.wait()
        for (n, _), ((x, res, ids, w, nw), y, h, hn) in zip(work, bufs):  # every kernel's first launch falls on all threads at once
            c.proj_forward([d], n, x, [y])
            c.moe_experts(dev, n, 3, x, ids, w, res, nw, h, hn)
        c.synchronize()
    except Exception as e:
        failed.append(e)

threads = [threading.Thread(target=body, args=a) for a in zip(contexts, streams, buffers)]
[t.start() for t in threads]
[t.join() for t in threads]
assert not failed, failed
for bufs in buffers:
    for (n, v), (_, y, h, hn) in zip(work, bufs):
        moe_ref.close(y.cpu().numpy(), *moe_ref.product(v[0], mat))
        check((h.cpu().numpy(), hn.cpu().numpy()), m, v[0], v[2], v[3], v[1], v[4])
[c.close() for c in contexts]
print("threads ok")
"""


def test_contexts_of_several_threads_begin_at_once():
    """A process of its own, so that the first launch of every kernel falls on four threads with a context each."""
    here = Path(__file__).resolve().parent
    r = subprocess.run([sys.executable, "-c", THREADS.format(path=[str(here), str(here.parent)])], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "threads ok" in r.stdout, r.stdout[-2000:] + r.stderr[-2000:]
