"""Trees of drafted tokens in float64, from the definitions: what a row sees, attention over a paged sequence, verification,
rows that are kept. Slow and plain; CPU tensors."""
import torch


def above(parents):
    """see [rows, rows] bool of one tree: a row sees itself and the rows above it; and the rows' depths."""
    n = len(parents)
    see, depth = torch.zeros(n, n, dtype=torch.bool), [0] * n
    for i, p in enumerate(parents):
        if 0 <= p < i:
            see[i], depth[i] = see[p], depth[p] + 1
        see[i, i] = True
    return see, depth


def words(see, n_words):
    """see [rows, m] as int64 words [rows, n_words]: bit j % 64 of word j / 64."""
    out = torch.zeros(see.shape[0], n_words, dtype=torch.int64)
    for i in range(see.shape[0]):
        for j in range(min(see.shape[1], 64 * n_words)):
            if see[i, j]:
                bit = 1 << (j % 64)
                out[i, j // 64] |= bit - (1 << 64) if bit >> 63 else bit
    return out


def attend(q, k, v, ok, see, scale):
    """q [rows, hq, d]: the last rows of a sequence with keys k, v [length, hkv, d], of which ok are there; see [rows, rows].
    Returns the outputs [rows, hq, d] and sum_j p_j |v_j| of each."""
    n, hq, d = q.shape
    length, hkv, _ = k.shape
    base = length - n
    out = torch.zeros(n, hq, d, dtype=torch.float64)
    size = torch.zeros_like(out)
    at = torch.arange(length)
    for i in range(n):
        new = at - base
        vis = ok & ((new < 0) | ((new >= 0) & (new <= i) & see[i, new.clamp(0, n - 1)]))
        if base + i < 0:
            vis = torch.zeros_like(ok)
        if not bool(vis.any()):
            continue
        kk, vv = k[vis], v[vis]
        for h in range(hkv):
            rep = hq // hkv
            p = torch.softmax(q[i, h * rep:(h + 1) * rep].double() @ kk[:, h].T * scale, -1)
            out[i, h * rep:(h + 1) * rep] = p @ vv[:, h]
            size[i, h * rep:(h + 1) * rep] = p @ vv[:, h].abs()
    return out, size


def softmax(x, t):
    """Shares of logits x [V] over temperature t: a NaN counts as -infinity, infinite logits (or, at an infinite
    temperature, all above -infinity) share alike; zeros for a row of nothing."""
    x = torch.where(x.isnan(), float("-inf"), x.double())
    top = x.max()
    if top == float("-inf"):
        return torch.zeros_like(x)
    if top == float("inf"):
        w = (x == top).double()
    elif t == float("inf"):
        w = (x > float("-inf")).double()
    else:
        w = torch.exp((x - top) / t)
    return w / w.sum()


def verify(logits, tokens, parents, u, r, t, depth, draft=None):
    """One tree: (path, next). What is left of a row's distribution is renormalised after each rejection."""
    V = logits.shape[1]
    path, node = [0], 0
    while True:
        x = logits[node].double()
        x = torch.where(x.isnan(), float("-inf"), x)
        best = int((x == x.max()).nonzero()[0]) if x.max() > float("-inf") else -1
        kids = [i for i in range(node + 1, len(parents)) if parents[i] == node] if len(path) < depth else []
        greedy = not t > 0
        left = None if greedy else softmax(logits[node], t)
        taken = None
        for i in kids:
            tok = int(tokens[i])
            if not 0 <= tok < V:
                if not greedy and draft is not None:           # a rejection all the same
                    left = _less(left, draft[node])
                continue
            if greedy:
                yes = tok == best
            elif draft is None:
                yes = float(u[i]) * float(left.sum()) < float(left[tok])
                if not yes:
                    left[tok] = 0
            else:
                yes = float(u[i]) * float(_share(draft[node])[tok]) * float(left.sum()) < float(left[tok])
                if not yes:
                    left = _less(left, draft[node])
            if yes:
                taken = i
                break
        if taken is None:
            break
        node = taken
        path.append(node)
    if greedy or best < 0:
        return path, best
    run = torch.cumsum(left, 0)
    if not float(run[-1]) > 0:
        return path, best
    over = (run > float(r) * float(run[-1])).nonzero()
    return path, int(over[0]) if len(over) else int((left > 0).nonzero()[-1])


def _share(q):
    q = q.double()
    return torch.where(q > 0, q, 0.0)


def _less(left, q):
    left = (left - _share(q)).clamp(min=0)
    return left / left.sum() if float(left.sum()) > 0 else left


def keep(path, count, rows):
    """The (from, to) rows that move: a path rises, and an entry that does not, or is no row, ends it."""
    out, before = [], -1
    for j in range(min(count, len(path), rows)):
        if not before < path[j] < rows:
            break
        before = path[j]
        out.append((path[j], j))
    return out
