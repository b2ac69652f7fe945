"""The mixture-of-experts operators in 64 bits, and the error bounds their tests use."""
import numpy as np

EPS = 2.0 ** -24  # half a step of fp32, relative


def weights(rng, out_dim, in_dim, lead=()):
    """A random 4-bit affine matrix (words uint32, scales and biases as bf16 bit patterns)."""
    w = rng.integers(0, 2 ** 32, size=(*lead, out_dim, in_dim // 8), dtype=np.uint64).astype(np.uint32)
    scales = bf16(rng.uniform(0.002, 0.008, size=(*lead, out_dim, in_dim // 64)))
    biases = bf16(-f32(scales) * (7.5 + 0.5 * rng.standard_normal(scales.shape)))
    return w, scales, biases


def spread(rng, mat, ratio):
    """The matrix with three of every four groups of 64 inputs scaled down by `ratio` (some of those to nothing but a bias)."""
    w, scales, biases = mat
    small = np.arange(scales.shape[-1]) % 4 != 1
    s, b = (np.where(small, f32(a) * ratio, f32(a)) for a in (scales, biases))
    s[..., small] *= rng.random(s[..., small].shape) > 0.1
    return w, bf16(s), bf16(b)


def bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def f32(bits):
    return (np.asarray(bits).astype(np.uint32) << 16).view(np.float32)


def parts(w, scales, biases):
    """nibbles, and scale and bias of each, as float64 [..., out, in]."""
    q = ((w[..., None] >> np.arange(0, 32, 4, dtype=np.uint32)) & 15).astype(np.float64).reshape(*w.shape[:-1], -1)
    return q, np.repeat(f32(scales).astype(np.float64), 64, -1), np.repeat(f32(biases).astype(np.float64), 64, -1)


def matrix(w, scales, biases):
    q, s, b = parts(w, scales, biases)
    return q * s + b


def product(x, mat):
    """(x W^T, bound of the error of computing it in fp32).

    Every output is a sum of in / 64 group terms s * N + b * X, N and X sums of 64 products that reach the tensor cores
    (or an integer sum) without rounding.  At most in / 64 + 64 roundings or truncations lie between a product and the
    output -- the additions over the groups and over the parts of a split row, the tensor cores' own 64-term sums, the
    conversions -- each off by half a step of fp32 relative to a sum that is no larger than that of the absolute terms."""
    q, s, b = parts(*mat)
    x = np.asarray(x, np.float64)
    a = np.abs(x)
    return x @ (q * s + b).T, (x.shape[-1] / 64 + 64) * EPS * (a @ (q * np.abs(s) + np.abs(b)).T)


def close(got, want, bound):
    """Elementwise within the bound, and in the 2-norm within what independent roundings of that size add up to: a bound of
    N worst-case steps comes to about sqrt(N) of them, and a single step is well below the absolute sum it is taken from."""
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape
    assert np.all(np.abs(got - want) <= bound), float((np.abs(got - want) / bound).max())
    norm = np.linalg.norm(want)
    if norm > 0:
        assert np.linalg.norm(got - want) <= 0.25 * np.linalg.norm(bound), (np.linalg.norm(got - want) / norm)


def route(logits, bias, rc):
    """ids, weights by the definition, in 64 bits (rc: a dict with FmRouteConfig's fields)."""
    E, k, G = rc["num_experts"], rc["top_k"], rc["num_groups"]
    ids = np.full((len(logits), k + rc["shared_expert"]), -1, np.int32)
    out = np.zeros(ids.shape)
    for t, row in enumerate(np.asarray(logits, np.float64)):
        x = row[:E]
        b = np.zeros(E) if bias is None else np.asarray(bias, np.float64)
        there = (x > -np.inf) & (b > -np.inf)
        if there.any():
            with np.errstate(over="ignore", invalid="ignore"):
                if rc["score"] == 0:
                    m = x[there].max()
                    s = np.where(there, np.where(x == m, 1.0, np.exp(x - m)), 0.0)
                    s = s / s.sum()
                else:
                    s = np.where(there, 1 / (1 + np.exp(-x)), 0.0)
            c = np.where(there, s + b, -np.inf)
            if rc["score"] == 0 and bias is None:
                key = np.where(there, x, -np.inf)  # the same order, without a tie by underflow
            else:
                key = c
            if G > 1:
                size = E // G
                total = np.full(G, -np.inf)
                for g in range(G):
                    v = np.sort((key if rc["group_best"] == 1 else c)[g * size:(g + 1) * size])[::-1][: rc["group_best"]]
                    if v[0] > -np.inf:
                        total[g] = v[v > -np.inf].sum()
                keep = np.argsort(-total, kind="stable")[: rc["top_groups"]]
                mask = np.isin(np.arange(E) // size, keep)
                key = np.where(mask, key, -np.inf)
            order = np.argsort(-key, kind="stable")[:k]
            order = order[key[order] > -np.inf]
            w = s[order]
            if rc["renormalize"] and len(order):
                # a common factor drops out; with it gone, scores that underflow even 64 bits keep their ratio
                v = x[order]
                log = v if rc["score"] == 0 else -np.logaddexp(0.0, -v)
                with np.errstate(invalid="ignore"):
                    w = np.where(log == log.max(), 1.0, np.exp(log - log.max()))
                w = w / w.sum()
            ids[t, : len(order)] = order
            out[t, : len(order)] = w * np.float64(np.float32(rc["scale"]))
        if rc["shared_expert"]:
            ids[t, k] = E
            with np.errstate(over="ignore"):
                out[t, k] = 1 / (1 + np.exp(-row[E]))
    return ids, out


def experts(gate, up, down, x, ids, weights, residual, norm_w, first=0, eps=1e-6):
    """(h, h_norm, bound of h): the stacks are (words, scales, biases) with a leading expert dimension.

    The bound follows the error through the chain: that of gate and up (product), SwiGLU's own few roundings (16 steps
    cover exp, the division and the products; |silu'| <= 1.1), the down product of the perturbed values, the weighted sum."""
    n, hidden = x.shape
    held = gate[0].shape[0]
    h = np.zeros((n, hidden)) if residual is None else np.asarray(residual, np.float64).copy()
    bound = np.abs(h) * 4 * EPS
    ids = np.asarray(ids, np.int64) - first
    for e in range(held):
        t, j = np.nonzero(ids == e)
        if len(t) == 0:
            continue
        g, bg = product(x[t], [m[e] for m in gate])
        u, bu = product(x[t], [m[e] for m in up])
        sil = g / (1 + np.exp(-g))
        a = sil * u
        ba = 1.1 * bg * np.abs(u) + np.abs(sil) * bu + 1.1 * bg * bu + 16 * EPS * np.abs(a)
        y, by = product(a, [m[e] for m in down])
        by = by + ba @ np.abs(matrix(*[m[e] for m in down])).T
        w = np.asarray(weights, np.float64)[t, j][:, None]
        np.add.at(h, t, w * y)
        np.add.at(bound, t, np.abs(w) * (by + (ids.shape[1] + 4) * EPS * np.abs(y)))
    inv = 1 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    nw = np.ones(hidden) if norm_w is None else f32(norm_w).astype(np.float64)
    return h, h * inv * nw, bound


def norm_bound(h, bound, norm_w, eps=1e-6):
    """Bound of h_norm's error: that of h, plus the relative error of the row's root mean square."""
    inv = 1 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    nw = np.ones(h.shape[1]) if norm_w is None else np.abs(f32(norm_w).astype(np.float64))
    rel = (np.abs(h) * bound).mean(1, keepdims=True) * inv ** 2 + (h.shape[1] / 256 + 32) * EPS
    return (bound + np.abs(h) * (rel + 8 * EPS)) * inv * nw
