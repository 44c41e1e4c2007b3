"""Plain restatements of the policy operators for the tests: sampling and loss
in 64 bits with numpy, and the AdamW step's 32-bit operations one by one."""
import numpy as np
import torch

FLT_MAX = float(np.finfo(np.float32).max)


def sample_row(x, mask, noise, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(action, logp, kept indices) of one row, from the definition."""
    x = np.asarray(x, np.float64)
    seen = x > -np.inf
    if mask is not None:
        seen &= np.asarray(mask) != 0
    seen = np.nonzero(seen)[0]
    if not len(seen):
        return -1, 0.0, seen
    x = np.minimum(x, FLT_MAX)
    order = seen[np.argsort(-x[seen], kind="stable")]
    if temperature <= 0:
        return order[0], 0.0, order[:1]
    with np.errstate(over="ignore"):
        d = (x[order] - x[order[0]]) / np.float64(temperature)
        e = np.exp(d)
    n = len(order) if top_k <= 0 else min(top_k, len(order))
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(e[:n])[:-1]])
        n = max(1, int((before < top_p * e[:n].sum()).sum()))
    n = max(1, int((e[:n] >= min(min_p, 1.0)).sum()))
    order, d, e = order[:n], d[:n], e[:n]
    s = d + (0.0 if noise is None else np.asarray(noise, np.float64)[order])
    s = np.where(np.isnan(s), -np.inf, s)
    best = np.lexsort((order, -s))[0]
    return order[best], float(d[best] - np.log(e.sum())), order


def sample(x, mask, noise, **kw):
    rows = len(x)
    pick = lambda v, i: v[i] if isinstance(v, np.ndarray) else v  # noqa: E731
    got = [sample_row(x[i], None if mask is None else mask[i], None if noise is None else noise[i],
                      **{k: pick(v, i) for k, v in kw.items()}) for i in range(rows)]
    return np.array([g[0] for g in got], np.int32), np.array([g[1] for g in got])


def loss(x, mask, target=None, label=None, weight=None, grad_scale=1.0):
    """(loss, grad, terms): terms[i] is the size of what a row's loss sums up."""
    x = np.asarray(x, np.float64)
    rows, actions = x.shape
    out, grad, terms = np.zeros(rows), np.zeros((rows, actions)), np.zeros(rows)
    for i in range(rows):
        seen = np.ones(actions, bool) if mask is None else np.asarray(mask[i]) != 0
        if not seen.any() or not (x[i][seen] > -np.inf).any():
            continue
        top = x[i][seen].max()
        d = np.where(seen, np.where(seen, x[i], 0.0) - top, -np.inf)
        e = np.exp(d)
        z = e.sum()
        if target is not None:
            t = np.where(seen, np.asarray(target[i], np.float64), 0.0)
        else:
            t = np.zeros(actions)
            if 0 <= label[i] < actions and seen[label[i]]:
                t[label[i]] = 1.0
        w = 1.0 if weight is None else float(weight[i])
        used = t != 0
        out[i] = w * (t.sum() * np.log(z) - (t[used] * d[used]).sum())
        terms[i] = abs(w) * (np.abs(t).sum() * (abs(np.log(z)) + 1) + np.abs(t[used] * d[used]).sum())
        grad[i] = np.where(seen, grad_scale * w * (e / z * t.sum() - t), 0.0)
    return out, grad, terms


def mix32(x):
    x = np.asarray(x, np.uint64) & np.uint64(0xFFFFFFFF)
    m = np.uint64(0xFFFFFFFF)
    x ^= x >> np.uint64(16)
    x = (x * np.uint64(0x7FEB352D)) & m
    x ^= x >> np.uint64(15)
    x = (x * np.uint64(0x846CA68B)) & m
    return x ^ (x >> np.uint64(16))


def to_8bit(x, u, nonzero):
    """One block of 256: (codes as the float values they stand for, scale).
    Exact arithmetic on numpy float32: the scale is a power of two."""
    most = np.max(np.abs(x[np.isfinite(x)]), initial=np.float32(0))
    k = 0
    if most > 0:
        f, e = np.frexp(most)  # most = f 2^e, f in [0.5, 1)
        k = max(int(e) - 1 - 8 + (1 if f > 0.875 else 0), -126)
    y = np.ldexp(np.abs(x), -k).astype(np.float32)
    with np.errstate(invalid="ignore"):
        e = np.maximum(np.frexp(y)[1] - 1, -6)
        q = np.floor((np.ldexp(y, 3 - e).astype(np.float32) + u.astype(np.float32)).astype(np.float32))
    if nonzero:
        q = np.where((q == 0) & (y > 0), np.float32(1), q)
    return np.copysign(np.ldexp(q, e - 3), x).astype(np.float32), np.float32(np.ldexp(1.0, k))


class AdamW:
    """The step in 32-bit operations, one numpy array per tensor (n rounded up
    to blocks in the states)."""

    def __init__(self, params, bits, lr, betas, eps, decays, scales, max_norm, seed):
        self.p = [np.array(p, np.float32).reshape(-1) for p in params]
        self.bits, self.lr, self.betas, self.eps, self.decays, self.scales = bits, lr, betas, eps, decays, scales
        self.max_norm, self.seed, self.t = max_norm, seed, 0
        pad = [-(-p.size // 256) * 256 for p in self.p]
        self.m = [np.zeros(k, np.float32) for k in pad]
        self.v = [np.zeros(k, np.float32) for k in pad]
        self.ms = [np.ones(k // 256, np.float32) for k in pad]
        self.vs = [np.ones(k // 256, np.float32) for k in pad]
        self.first = np.concatenate([[0], np.cumsum(pad)])

    def step(self, grads, grad_scale=1.0, coef=None):
        """coef: the clipping factor (float32) when max_norm is in use."""
        f = np.float32
        self.t += 1
        b1, b2 = self.betas
        key = int(mix32((self.t * 0x9E3779B9 + self.seed) & 0xFFFFFFFF))
        scale = f(grad_scale) * (f(1) if coef is None else f(coef))
        for k, g in enumerate(grads):
            if g is None:
                continue
            n, p = self.p[k].size, self.p[k]
            g = np.asarray(g, f).reshape(-1) * scale
            m, v = self.m[k][:n], self.v[k][:n]
            if self.bits == 8:
                m = m * np.repeat(self.ms[k], 256)[:n]
                r = v * np.repeat(self.vs[k], 256)[:n]
                v = r * r
            m = m * f(b1) + g * f(1 - b1)
            v = v * f(b2) + (g * g) * f(1 - b2)
            root = np.sqrt(v)
            decay = f(1 - self.lr * self.scales[k] * self.decays[k])
            step = f(self.lr / (1 - b1**self.t) * self.scales[k])
            correct = f(1 / np.sqrt(1 - b2**self.t))
            self.p[k] = p * decay - m / (root * correct + f(self.eps)) * step
            if self.bits == 32:
                self.m[k][:n], self.v[k][:n] = m, v
                continue
            pad = self.m[k].size
            at = np.arange(pad, dtype=np.uint64) + np.uint64(self.first[k])
            h = mix32((at + np.uint64(key)) & np.uint64(0xFFFFFFFF))
            um, uv = (h & np.uint64(0xFFFF)).astype(f) * f(2**-16), (h >> np.uint64(16)).astype(f) * f(2**-16)
            m, root = np.pad(m, (0, pad - n)), np.pad(root, (0, pad - n))
            for b in range(pad // 256):
                to = slice(256 * b, 256 * b + 256)
                self.m[k][to], self.ms[k][b] = to_8bit(m[to], um[to], False)
                self.v[k][to], self.vs[k][b] = to_8bit(root[to], uv[to], True)


def gumbel(shape, seed):
    return -torch.log(torch.empty(shape).exponential_(generator=torch.Generator().manual_seed(seed)))
