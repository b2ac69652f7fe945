"""The 64-bit reference of the mixture-of-experts tests against the CPU oracle, and the structs' ctypes mirrors (no GPU)."""
import re
from pathlib import Path

import numpy as np

import moe_ref

ROOT = Path(__file__).resolve().parents[1]


def test_product_is_the_oracles(port):
    rng = np.random.default_rng(0)
    m = moe_ref.weights(rng, 40, 512)
    x = rng.standard_normal((3, 512)).astype(np.float32)
    want, _ = port.out_proj_norm(*m, x, None, moe_ref.bf16(np.ones(40)))
    got, bound = moe_ref.product(x, m)
    assert np.abs(got - want).max() <= 1e-4 * np.abs(want).max()
    assert np.all(bound < 5e-4 * np.abs(want).max())


def test_bf16_helpers_round_trip():
    bits = np.arange(0, 0x7F80, 7, dtype=np.uint16)
    assert np.array_equal(moe_ref.bf16(moe_ref.f32(bits)), bits)


def test_routing_by_hand():
    rc = dict(num_experts=4, top_k=2, score=0, num_groups=2, top_groups=1, group_best=2, renormalize=1, scale=2.0, shared_expert=1)
    logits = np.log([[0.4, 0.05, 0.3, 0.25, 1.0]])  # group 1 (0.55) beats group 0 (0.45) although expert 0 is the best one
    ids, w = moe_ref.route(logits, None, rc)
    assert ids.tolist() == [[2, 3, 4]]
    assert np.allclose(w, [[2 * 0.3 / 0.55, 2 * 0.25 / 0.55, 0.5]])


def test_structs_match_the_header(pkg):
    text = (ROOT / "include" / "fm_attn.h").read_text()
    for name in ("FmRouteConfig", "FmExpertWeights", "FmProjWeights"):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = [f.strip(" *") for line in re.findall(r"\b(?:int|float|int64_t|const uint32_t|const uint16_t)\s+([^;]+);", body) for f in line.split(",")]
        assert fields == [f[0] for f in getattr(pkg.binding, name)._fields_]


def test_default_route_config(pkg):
    rc = pkg.route_config(top_k=8)
    assert (rc.num_experts, rc.top_k, rc.score, rc.num_groups, rc.top_groups, rc.group_best, rc.renormalize, rc.scale, rc.shared_expert) == (512, 8, 0, 1, 1, 1, 1, 1.0, 0)
