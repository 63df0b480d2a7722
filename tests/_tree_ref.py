"""Plain 64-bit forms of the tree-speculation operators, node by node."""
import torch


def way_up(row, i):
    """Nodes from the root down to i, or [] for padding."""
    out = []
    while True:
        out.append(i)
        p = row[i]
        if p == -1:
            return out[::-1]
        if not 0 <= p < i:
            return []
        i = p


def random_tree(rng, S, kind):
    if kind == "chain":
        return list(range(-1, S - 1))
    if kind == "star":
        return [-1] + [0] * (S - 1)
    if kind == "roots":  # several nodes directly below the cached positions
        return [-1 if rng.random() < 0.3 else rng.randrange(i) if i else -1 for i in range(S)]
    row = [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, S)]
    if kind == "padded":
        for i in range(1, S):
            if rng.random() < 0.2:
                row[i] = rng.choice((-2, -7, i, i + 1, 300, 2 ** 31 - 1, -2 ** 31))
    return row


def attention(q, kt, v, rows, lens):
    """q [B, nkv, rep * S, hd] -> (out, sum p |v|, max |q| |k|) [B, S, nkv * rep, hd], float64 on
    q's device; rows: a tree per sequence."""
    B, nkv, R, hd = q.shape
    S = len(rows[0])
    rep = R // S
    out = torch.zeros(B, S, nkv * rep, hd, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    big = 0.0
    for b in range(B):
        C = int(lens[b])
        if C < 0:
            continue
        for i in range(S):
            way = way_up(rows[b], i)
            if not way:
                continue
            at = torch.tensor(list(range(C)) + [C + a for a in way], device=q.device)
            for g in range(nkv):
                k = kt[b, g].double().index_select(1, at)
                vv = v[b, g].double().index_select(0, at)
                qq = q[b, g].double().view(rep, S, hd)[:, i]
                p = torch.softmax(qq @ k * hd ** -0.5, -1)
                out[b, i, g * rep:(g + 1) * rep] = p @ vv
                mag[b, i, g * rep:(g + 1) * rep] = p @ vv.abs()
                big = max(big, float((qq.abs() @ k.abs()).nan_to_num(0, 0, 0).max()))
    return out, mag, big * hd ** -0.5


def append(qkv, cos, sin, rows, lens, nh, kt, v):
    """(q [B, nkv, rep * S, hd], kt, v) in float64; kt, v: copies of the cache."""
    B, nkv, hd, n = kt.shape
    S, rep = len(rows[0]), nh // nkv
    kt, v = kt.double().clone(), v.double().clone()
    q = torch.zeros(B, nkv, rep, S, hd, dtype=torch.float64, device=qkv.device)
    x = qkv.double().view(B, S, nh + 2 * nkv, hd)
    for b in range(B):
        C = int(lens[b])
        for i in range(S):
            way = way_up(rows[b], i)
            if C < 0 or not way:
                continue
            P = C + len(way) - 1
            if P >= cos.shape[0] or C + i >= n:
                q[b, :, :, i] = float("nan")
                continue
            for h in range(nh + nkv):
                a = x[b, i, h]
                rh = torch.cat((-a[hd // 2:], a[:hd // 2]))
                y = a * cos[P].double() + rh * sin[P].double()
                if h < nh:
                    q[b, h // rep, h % rep, i] = y
                else:
                    kt[b, h - nh, :, C + i] = y
                    v[b, h - nh, C + i] = x[b, i, h + nkv]
    return q.view(B, nkv, rep * S, hd), kt, v


def verify(logits, tokens, rows, u, draft, temps):
    """(path, count, token) as lists, by the definition: residuals normalised one after the
    other."""
    B, S, V = logits.shape
    paths, toks, margin = [], [], 1.0
    for b in range(B):
        t = float(temps[b])

        def soft(x):
            x = torch.where(x.isnan(), -torch.inf, x.double()).clamp(max=3.4028234663852886e38)
            if x.max() == -torch.inf:
                return torch.zeros_like(x)
            if t <= 0:
                y = torch.zeros_like(x)
                y[int((x == x.max()).nonzero()[0])] = 1
                return y
            e = torch.exp((x - x.max()) / t)
            return e / e.sum()

        got = [0]
        while True:
            n = got[-1]
            p = soft(logits[b, n])
            r, done, mass = p, True, 1.0
            for i in range(n + 1, S):
                if rows[b][i] != n or not way_up(rows[b], i):
                    continue
                x = int(tokens[b, i])
                if not 0 <= x < V:
                    continue
                if draft is not None and t > 0:
                    q = soft(draft[b, n])
                else:
                    q = torch.zeros_like(p)
                    q[x] = 1
                a, bnd = float(r[x]), float(u[b, i]) * float(q[x])
                if t > 0 and a != bnd:
                    margin = min(margin, abs(a - bnd) / max(a, bnd))
                if (a > 0 if t <= 0 else bnd < a):
                    got.append(i)
                    done = False
                    break
                if t > 0:
                    left = (r - q).clamp(min=0)
                    mass *= float(left.sum())
                    if mass <= 2.0 ** -40:
                        r = p
                        break
                    r = left / left.sum()
            if done:
                break
        paths.append(got)
        pos = (r > 0).nonzero().flatten().tolist()
        run = r.cumsum(0)
        hit = ((run > float(u[b, 0]) * float(run[-1])) & (r > 0)).nonzero().flatten().tolist()
        toks.append(hit[0] if hit else pos[-1] if pos else -1)
    return paths, toks, margin
