"""The operators for experts outside a stack, stated in 64 bits with numpy, for the tests of salt_b200_route_experts, _mxfp4_* and
_combine_experts."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def scale_pitch(cols):
    return (cols // 32 + 15) // 16 * 16


def mx_quantize(x):
    """Rows of any float type -> (E2M1 codes [rows][cols] one per byte, E8M0 bytes [rows][cols / 32])."""
    b = np.asarray(x, np.float64).reshape(x.shape[0], -1, 32)
    with np.errstate(invalid="ignore"):
        top = np.abs(b).max(axis=2)
        bad = ~np.isfinite(b).all(axis=2)
    exponent = np.frexp(np.where(bad | (top == 0), 1.0, top))[1] - 1          # floor(log2), exact
    byte = np.where(top == 0, 0, np.clip(exponent - 2 + 127, 0, 254))
    u = np.where(bad[:, :, None], 0.0, b) / np.exp2(byte.astype(np.float64) - 127)[:, :, None]
    a = np.minimum(np.abs(u), 6.0)
    distance = np.abs(a[..., None] - GRID)
    # the nearest point; of two equally near ones the even code
    code = np.argmin(distance + np.where(np.arange(8) % 2, 1e-9, 0.0), axis=-1).astype(np.uint8)
    code |= (np.signbit(u).astype(np.uint8) << 3)
    code[bad] = 0
    return code.reshape(x.shape), np.where(bad, 255, byte).astype(np.uint8)


def mx_pack(code):
    return (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)


def mx_unpack(packed):
    return np.stack((packed & 15, packed >> 4), axis=-1).reshape(*packed.shape[:-1], -1)


def mx_values(code, byte):
    v = GRID[code & 7] * np.where(code & 8, -1.0, 1.0)
    with np.errstate(invalid="ignore"):
        s = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
        return v * np.repeat(s, 32, axis=-1)


def act(name, g):
    if name == "silu":
        return g / (1 + np.exp(-g))
    return 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)))


HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}       # half a step, relative to the value
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}    # the smallest step


def product(xv, wv):
    """(y, bound on a 32-bit sum's error): xv [n][K], wv [R][K].  A sum of K / 64 steps (or, per lane, of K / 32 blocks), each of which
    rounds or cuts off at most one unit of 2^-23 of what has been added so far, twice that for the products' alignment."""
    with np.errstate(invalid="ignore"):
        return xv @ wv.T, (xv.shape[1] / 32 + 8) * 2.0 ** -23 * (np.abs(xv) @ np.abs(wv).T)


def gated(name, xv, gate, up):
    g, eg = product(xv, gate)
    u, eu = product(xv, up)
    # slope of either function below 1.13; evaluation in 32 bits within 2^-21 of the argument
    with np.errstate(over="ignore"):
        return act(name, g) * u, (1.13 * eg + 2.0 ** -21 * np.abs(g)) * (np.abs(u) + eu) + np.abs(act(name, g)) * eu


def close(got, want, err, dtype, what=""):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, what
    nan = np.isnan(want)
    assert (np.isnan(got) == nan).all(), f"{what}: NaN in other places"
    limit = err + HALF[dtype] * (np.abs(want) + err) + TINY[dtype]
    off = np.abs(got - want) - limit
    off[nan] = -1
    if (off > 0).any():
        i = np.unravel_index(np.argmax(off), off.shape)
        raise AssertionError(f"{what}: {int((off > 0).sum())} of {off.size} outside; worst at {i}: {got[i]!r} against {want[i]!r}, "
                             f"{abs(got[i] - want[i]):.3e} where {limit[i]:.3e} is allowed")


def route(logits, topk, scoring="softmax", bias=None, n_groups=1, topk_groups=1, group_top=1, renormalize=True, scale=1.0):
    """One token after the other -> (selected, weights), the last places -1 and 0."""
    T, E = logits.shape
    ids, weights = np.full((T, topk), -1, np.int32), np.zeros((T, topk))
    for t in range(T):
        l = np.asarray(logits[t], np.float64)
        live = ~np.isnan(l) & (l > -np.inf)
        s = np.zeros(E)
        with np.errstate(over="ignore", invalid="ignore"):
            if scoring == "sigmoid":
                s[live] = np.where(l[live] >= 0, 1 / (1 + np.exp(-np.abs(l[live]))), np.exp(-np.abs(l[live])) / (1 + np.exp(-np.abs(l[live]))))
            elif live.any():
                m = l[live].max()
                p = np.where(l[live] == m, 1.0, np.exp(l[live] - m))
                s[live] = p / p.sum()
        key = l.copy() if bias is None else s + np.asarray(bias, np.float64)
        live &= ~np.isnan(key) & (key > -np.inf)
        if n_groups > 1:
            per, rank = E // n_groups, []
            for g in range(n_groups):
                e = [i for i in range(g * per, (g + 1) * per) if live[i]]
                if e:
                    # without a bias and with one key the logit orders the groups as the score does
                    value = key if bias is not None or group_top == 1 else s
                    rank.append((-sum(sorted((value[i] for i in e), reverse=True)[:group_top]), g))
            stay = {g for _, g in sorted(rank)[:topk_groups]}
            live &= np.array([i // per in stay for i in range(E)])
        best = sorted(sorted(np.nonzero(live)[0], key=lambda i: (-key[i], i))[:topk])
        w = s[best]
        if renormalize and w.sum() > 0:
            w = w / w.sum()
        ids[t, :len(best)], weights[t, :len(best)] = best, scale * w
    return ids, weights


def grouping(ids, n_experts):
    flat = ids.reshape(-1)
    order = [i for e in range(n_experts) for i in np.nonzero(flat == e)[0]]
    g2c, c2g = np.full(flat.size, -1, np.int32), np.full(flat.size, -1, np.int32)
    g2c[:len(order)] = order
    c2g[order] = np.arange(len(order))
    counts = np.array([(flat == e).sum() for e in range(n_experts)])
    return np.concatenate(([0], np.cumsum(counts))).astype(np.int32), g2c, c2g
