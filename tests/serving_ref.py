"""Plain 64-bit forms of the serving-step operators (numpy), and the batches their tests run on."""
import numpy as np

NP = {"f32": np.float32, "f16": np.float16}


def torch_dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def f64(t):
    return t.detach().cpu().double().numpy()


class Batch:
    """Sequences with `lens` entries, `counts` of them new, over shuffled pages of a pool with spare ones."""

    def __init__(self, lens, counts, kv_heads, hd, page, kv, seed=0, book=False, spare_pages=2, values=True):
        import torch
        self.lens, self.counts, self.kv_heads, self.hd, self.page, self.kv = list(lens), list(counts), kv_heads, hd, page, kv
        g = torch.Generator("cpu").manual_seed(seed)
        need = [-(-n // page) for n in lens]
        total, most = sum(need) + spare_pages, max(need + [1]) + 1
        ids = torch.randperm(total, generator=g).to(torch.int32)
        table = torch.full((len(lens), most), -7, dtype=torch.int32)  # places past a sequence's pages name none
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = ids[at:at + n]
            at += n
        pool = torch.randn(total, 2, kv_heads, page, hd, generator=g) if values else torch.zeros(total, 2, kv_heads, page, hd)
        self.pool = pool.to(torch_dtype(kv)).cuda()
        self.table = table.cuda()
        self.tlens = torch.tensor(self.lens, dtype=torch.int32).cuda()
        self.starts = np.concatenate([[0], np.cumsum(self.counts)]).astype(np.int32)
        self.row_start = torch.from_numpy(self.starts).cuda()
        self.rows, self.cap = int(self.starts[-1]), most * page
        self.weight = self.position = None
        if book:
            self.weight = torch.exp(torch.randn(len(lens), kv_heads, self.cap, generator=g)).cuda()
            self.position = (3 * torch.arange(self.cap, dtype=torch.int32)).expand(len(lens), kv_heads, self.cap).contiguous().cuda()
        self.g = g

    def normal(self, *shape, dtype="f32"):
        import torch
        return torch.randn(*shape, generator=self.g).to(torch_dtype(dtype)).cuda()

    def cache(self):
        from rustane_b200 import ops
        return ops.PagedCache(self.pool, self.table, self.tlens, self.weight, self.position)

    def entries(self, b, which, pool=None):
        """[kv_heads, lens[b], hd] in 64 bits."""
        n = self.lens[b]
        pages = self.table[b, : -(-n // self.page)].long()
        x = (self.pool if pool is None else pool)[pages][:, which]
        return f64(x).transpose(1, 0, 2, 3).reshape(self.kv_heads, -1, self.hd)[:, :n]


def attention(batch, q, scale=None, window=0):
    """(out, lse, sum of |p v|, what each entry got [b][kv_heads, len], largest sum of |q k| scale) of every row."""
    hd, kv = batch.hd, batch.kv_heads
    q = f64(q)
    rows, heads = q.shape[:2]
    group, scale = heads // kv, hd ** -0.5 if scale is None else scale
    out, mass, lse, got, worst = np.zeros_like(q), np.zeros_like(q), np.full((rows, heads), -np.inf), [], 0.0
    for b, n in enumerate(batch.lens):
        k, v = batch.entries(b, 0), batch.entries(b, 1)
        got.append(np.zeros((kv, n)))
        for j in range(batch.counts[b]):
            r, last = batch.starts[b] + j, n - batch.counts[b] + j
            first = max(0, last + 1 - window) if window else 0
            if last < first:
                continue
            for h in range(heads):
                kk, vv = k[h // group, first:last + 1], v[h // group, first:last + 1]
                s = kk @ q[r, h] * scale
                worst = max(worst, float((np.abs(kk) @ np.abs(q[r, h])).max() * scale))
                top = s.max()
                p = np.exp(s - top)
                lse[r, h] = top + np.log(p.sum())
                p /= p.sum()
                out[r, h], mass[r, h] = p @ vv, p @ np.abs(vv)
                got[b][h // group, first:last + 1] += p
    return out, lse, mass, got, worst


def rotate(x, positions, freq, magnitude, layout):
    """x [rows, heads, hd] (64 bits), freq [rot / 2] radians a position."""
    rot = 2 * len(freq)
    a = np.asarray(positions, dtype=np.float64)[:, None] * freq
    c, s = np.cos(a)[:, None] * magnitude, np.sin(a)[:, None] * magnitude
    y = x.copy()
    u, w = (x[..., :rot // 2], x[..., rot // 2:rot]) if layout == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
    if layout == "half":
        y[..., :rot // 2], y[..., rot // 2:rot] = u * c - w * s, u * s + w * c
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = u * c - w * s, u * s + w * c
    return y


def frequencies(rot, base, scaling, factor, original):
    i = np.arange(rot // 2, dtype=np.float64)
    if scaling == "ntk" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f, magnitude = base ** (-2.0 * i / rot), 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        def where(turns):
            return rot * np.log(original / (turns * 2 * np.pi)) / (2 * np.log(base))
        low, high = max(np.floor(where(32.0)), 0), min(np.ceil(where(1.0)), rot - 1)
        ramp = np.clip((i - low) / max(high - low, 0.001), 0, 1)
        f, magnitude = f / factor * ramp + f * (1 - ramp), 0.1 * np.log(factor) + 1
    return f, magnitude


def evict(weight, position, n, keep, sinks, recent):
    """Moves [(to, from)] of one head of n entries."""
    if n <= keep:
        return []
    newest = int(position[:n].max())
    order = sorted(range(n), key=lambda i: (not (position[i] < sinks or position[i] > newest - recent),
                                             np.isnan(weight[i]), -weight[i] if not np.isnan(weight[i]) else 0.0, i))
    stay = set(order[:keep])
    return list(zip([i for i in range(keep) if i not in stay], [i for i in range(keep, n) if i in stay]))


def softmax(x):
    x = np.asarray(x, dtype=np.float64)
    e = np.exp(x - x.max())
    return e / e.sum()


def verify(target, draft, tokens, uniforms, draws, starts, temperature):
    """(accepted, out tokens) of a batch; logits as 64-bit arrays."""
    accepted, out = [], []
    for b in range(len(starts) - 1):
        r0, n = int(starts[b]), int(starts[b + 1] - starts[b])
        got, extra = [], None
        for j in range(n):
            t = target[r0 + j]
            bad = np.isnan(t).any() or not np.isfinite(t.max())
            x = int(tokens[r0 + j + 1]) if j < n - 1 else None
            if bad:
                extra = -1
            elif temperature == 0:
                best = int(t.argmax())
                if x == best:
                    got.append(x)
                    continue
                extra = best
            else:
                p, left = softmax(t / temperature), None
                if x is not None:
                    if draft is None:
                        q = np.zeros_like(p)
                        if 0 <= x < len(p):
                            q[x] = 1.0
                        qx = 1.0
                    else:
                        d = draft[r0 + j]
                        if np.isnan(d).any() or not np.isfinite(d.max()):
                            extra = -1
                            break
                        q = softmax(d / temperature)
                        qx = q[x] if 0 <= x < len(p) else 1.0
                    if 0 <= x < len(p) and uniforms[r0 + j] * qx < p[x]:
                        got.append(x)
                        continue
                    left = np.maximum(p - q, 0)
                sums = np.cumsum(p if left is None or left.sum() <= 0 else left)
                extra = int(np.searchsorted(sums, draws[b] * sums[-1], side="right"))
            break
        accepted.append(len(got))
        if n:
            out += got + [extra] + [-1] * (n - len(got) - 1)
    return np.array(accepted), np.array(out)
