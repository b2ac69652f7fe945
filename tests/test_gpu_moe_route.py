"""fm_moe_route against its definition in 64 bits: ids exactly, weights to fp32."""
import numpy as np
import pytest
import torch

import moe_ref
from test_gpu_proj_forward import context

pytestmark = pytest.mark.gpu
BASE = dict(num_experts=64, top_k=4, score=0, num_groups=1, top_groups=1, group_best=1, renormalize=1, scale=1.0, shared_expert=0)


def run(pkg, c, rc, logits, bias=None):
    n, slots = len(logits), rc["top_k"] + rc["shared_expert"]
    dev = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda()  # noqa: E731
    ids = torch.full((n + 1, slots), 77, device="cuda", dtype=torch.int32)
    w = torch.full((n + 1, slots), 77.0, device="cuda")
    c.moe_route(pkg.route_config(**rc), n, dev(logits), dev(bias), ids, w)
    c.synchronize()
    assert torch.all(ids[n:] == 77) and torch.all(w[n:] == 77.0)
    return ids[:n].cpu().numpy(), w[:n].cpu().numpy()


def check(got, want):
    """Weights: exp and the sigmoid to 2 ulp and the exponent's own rounding (2^-24 of it, exponents up to 40 here), the sum
    over the experts, two divisions, the factor: 128 half steps cover them."""
    assert np.array_equal(got[0], want[0])
    assert np.all(np.abs(got[1] - want[1]) <= 128 * moe_ref.EPS * np.abs(want[1]) + 1e-37)


CASES = [dict(), dict(num_experts=512, top_k=10), dict(num_experts=512, top_k=10, shared_expert=1), dict(num_experts=1, top_k=1),
         dict(num_experts=33, top_k=32), dict(num_experts=32, top_k=32, renormalize=0), dict(num_experts=1000, top_k=3, scale=2.5), dict(num_experts=1024, top_k=17, score=1),
         dict(num_experts=256, top_k=8, score=1, num_groups=8, top_groups=4, group_best=2, scale=2.5), dict(num_experts=100, top_k=6, num_groups=5, top_groups=2, renormalize=0),
         dict(num_experts=60, top_k=7, num_groups=4, top_groups=2, group_best=2), dict(num_experts=32, top_k=3, num_groups=32, top_groups=3, group_best=2),
         dict(num_experts=96, top_k=9, score=1, num_groups=3, top_groups=3, group_best=1, renormalize=0, shared_expert=1)]


@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_random_logits(pkg, case, with_bias):
    rc = {**BASE, **case}
    rng = np.random.default_rng(rc["num_experts"] + rc["top_k"])
    c = context(pkg, max_batch=512)
    for n in (1, 3, 130):
        logits = (2.0 * rng.standard_normal((n, rc["num_experts"] + rc["shared_expert"]))).astype(np.float32)
        bias = (0.1 * rng.standard_normal(rc["num_experts"])).astype(np.float32) if with_bias else None
        check(run(pkg, c, rc, logits, bias), moe_ref.route(logits, bias, rc))
    c.close()


@pytest.mark.parametrize("score", [0, 1])
def test_borders_that_fp32_cannot_decide(pkg, score):
    """Scores that differ by less than fp32's rounding of them, and equal ones: 64 bits decide, ties go to the lowest index."""
    rc = {**BASE, "num_experts": 128, "top_k": 8, "score": score}
    rng = np.random.default_rng(4)
    logits = (3.0 + 1e-6 * rng.integers(-3, 4, size=(64, 128))).astype(np.float32)
    logits[:, ::5] -= 9.0
    logits[32:, 7] = logits[32:, 90]
    bias = (1e-8 * rng.integers(-2, 3, size=128)).astype(np.float32)
    grouped = {**rc, "num_groups": 8, "top_groups": 3, "group_best": 2}
    c = context(pkg)
    for r in (rc, grouped):
        for b in (None, bias):
            check(run(pkg, c, r, logits, b), moe_ref.route(logits, b, r))
    same = np.zeros((3, 128), np.float32)
    for r in (rc, grouped):
        ids, w = run(pkg, c, r, same)
        assert np.array_equal(ids, np.tile(np.arange(8, dtype=np.int32), (3, 1))) and np.allclose(w, 1 / 8, rtol=1e-6, atol=0)
    c.close()


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("experts,groups", [(256, 8), (512, 8), (256, 4), (1024, 32), (120, 5), (18, 6)])
def test_groups_that_fp32_cannot_order(pkg, score, best, experts, groups):
    """Rows whose groups' best choices lie closer than fp32 tells, beside ordinary ones; whole and part registers per group."""
    rc = {**BASE, "num_experts": experts, "top_k": 3, "score": score, "num_groups": groups, "top_groups": groups // 2, "group_best": best}
    rng = np.random.default_rng(experts + groups)
    logits = rng.standard_normal((48, experts)).astype(np.float32)
    tight = (2.0 + 1e-6 * rng.integers(-2, 3, size=(24, experts))).astype(np.float32)
    logits[::2] = np.where(rng.random((24, experts)) < 0.3, tight, logits[::2] - 3.0)
    logits[4:12, : experts // groups] = -np.inf  # a group without an expert
    bias = (1e-7 * rng.standard_normal(experts)).astype(np.float32)
    c = context(pkg)
    for b in (None, bias):
        check(run(pkg, c, rc, logits, b), moe_ref.route(logits, b, rc))
    c.close()


def rows_of_close_logits_far_below_the_best(rng, experts):
    """More than 32 logits that share all but the last bits, beside larger ones whose distance leaves them without a score."""
    up = np.arange(experts) * 2.0 ** -23
    rows = np.zeros((8, experts), np.float32)
    rows[0] = 1.0 + up; rows[0, 0] = 1000.0
    rows[1] = 1.0 + up; rows[1, 3] = np.inf
    rows[2] = 1.0 + up[rng.permutation(experts)]; rows[2, experts // 2] = 800.0
    rows[3] = np.arange(experts) * 2.0 ** -149; rows[3, 1] = 1.0   # numbers that are lost beside the largest
    for row, mask in ((4, -1e4), (5, -1e5), (6, -3e38)):            # a mask that is added and finite, few experts without it
        rows[row] = rng.standard_normal(experts) + (mask if row < 6 else 0)
        rows[row] = rows[row] if row < 6 else mask
        free = rng.permutation(experts)[:2]
        rows[row, free] = rng.standard_normal(2)
    rows[7] = -2000.0 + up; rows[7, :5] = np.nan; rows[7, 9] = 0.0
    return rows


@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("experts", [64, 256, 512, 1024])
def test_softmax_without_a_bias_goes_by_the_logits(pkg, experts, groups):
    """However far below the largest logit the border lies: there are no ties by underflow."""
    rng = np.random.default_rng(experts + groups)
    logits = rows_of_close_logits_far_below_the_best(rng, experts)
    c = context(pkg)
    for top in (3, 10, 32 if experts > 64 else 16):
        for renorm in (0, 1):
            rc = {**BASE, "num_experts": experts, "top_k": top, "num_groups": groups, "top_groups": max(1, groups - 1), "renormalize": renorm}
            check(run(pkg, c, rc, logits), moe_ref.route(logits, None, rc))
    c.close()


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("experts,groups", [(32, 4), (256, 8), (512, 8), (60, 6)])
def test_groups_whose_choices_cancel(pkg, score, experts, groups):
    """A group's best two add up to about 1 while each is a thousand: their roundings are those of the thousands."""
    rc = {**BASE, "num_experts": experts, "top_k": 2, "score": score, "num_groups": groups, "top_groups": groups // 2, "group_best": 2}
    rng = np.random.default_rng(experts + score)
    logits = (1e-3 * rng.standard_normal((64, experts))).astype(np.float32)
    bias = np.full(experts, -1000.0, np.float32)
    bias[:: experts // groups] = 1000.0
    c = context(pkg)
    check(run(pkg, c, rc, logits, bias), moe_ref.route(logits, bias, rc))
    c.close()


@pytest.mark.parametrize("experts,groups", [(32, 4), (256, 8), (512, 8), (60, 6)])
def test_groups_whose_scores_are_subnormal(pkg, experts, groups):
    """Two experts of one group hold all of the weight, the others' scores are a few of fp32's smallest steps."""
    rc = {**BASE, "num_experts": experts, "top_k": 6, "num_groups": groups, "top_groups": 2, "group_best": 2}
    rng = np.random.default_rng(experts)
    logits = (-99.0 + 0.05 * rng.standard_normal((64, experts))).astype(np.float32)
    logits[:, :2] += 99.0
    logits[:, 2: experts // groups] = -np.inf
    c = context(pkg)
    check(run(pkg, c, rc, logits), moe_ref.route(logits, None, rc))
    c.close()


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("groups", [1, 4])
def test_experts_that_are_not_available(pkg, score, groups):
    rc = {**BASE, "num_experts": 40, "top_k": 6, "score": score, "num_groups": groups, "top_groups": min(groups, 2), "group_best": 2, "shared_expert": 1}
    rng = np.random.default_rng(6)
    logits = rng.standard_normal((12, 41)).astype(np.float32)
    logits[0, :40] = -np.inf                       # nothing is left
    logits[1, :40] = -np.inf; logits[1, [5, 33]] = 0.5, 0.25
    logits[2, 3:37] = np.nan
    logits[3, :40] = np.finfo(np.float32).min      # the lowest finite value is a logit like any other
    logits[4, 1:40] = np.finfo(np.float32).min
    logits[5, [4, 9]] = np.inf
    logits[6, 40] = -np.inf
    logits[7, :40] = -200.0 + 0.5 * rng.standard_normal(40)
    logits[8, 10:30] = -np.inf
    bias = (0.1 * rng.standard_normal(40)).astype(np.float32)
    bias[[2, 11]] = -np.inf, np.nan
    c = context(pkg)
    for b in (None, bias):
        for renorm in (0, 1):
            r = {**rc, "renormalize": renorm}
            check(run(pkg, c, r, logits, b), moe_ref.route(logits, b, r))
    c.close()


def test_host_pointers(pkg):
    rc = {**BASE, "shared_expert": 1}
    rng = np.random.default_rng(1)
    logits = rng.standard_normal((9, 65)).astype(np.float32)
    c = context(pkg, host=True)
    ids, w = np.empty((9, 5), np.int32), np.empty((9, 5), np.float32)
    c.moe_route(pkg.route_config(**rc), 9, logits, None, ids, w)
    check((ids, w), moe_ref.route(logits, None, rc))
    c.close()


def test_refusals(pkg):
    c = context(pkg, max_batch=4)
    x = torch.zeros((8, 64), device="cuda")
    ids, w = torch.zeros((8, 4), device="cuda", dtype=torch.int32), torch.zeros((8, 4), device="cuda")
    B = pkg.binding

    def status(n=1, args=(x, None, ids, w), **kw):
        with pytest.raises(pkg.FmError) as e:
            c.moe_route(pkg.route_config(**{**BASE, **kw}), n, *args)
        assert e.value.text.startswith("fm_moe_route")
        return e.value.status
    for bad in (dict(num_experts=0), dict(num_experts=1025), dict(top_k=0), dict(top_k=33), dict(num_groups=0), dict(num_groups=64), dict(top_k=32, shared_expert=1)):
        assert status(**bad) == B.FM_ERR_UNSUPPORTED
    for bad in (dict(score=2), dict(top_k=5, num_groups=16, top_groups=1), dict(num_groups=3), dict(top_groups=2), dict(top_groups=0),
                dict(num_groups=8, top_groups=2, group_best=3), dict(shared_expert=2), dict(n=5), dict(n=-1), dict(scale=float("nan"))):
        assert status(**bad) == B.FM_ERR_INVALID
    assert status(args=(None, None, ids, w)) == B.FM_ERR_INVALID and status(args=(x, None, None, w)) == B.FM_ERR_INVALID
    c.moe_route(pkg.route_config(**BASE), 0, x, None, ids, w)
    c.close()
