"""Plain forms of the operators over pages, in 64 bits and apart from any kernel, shared by
their tests: pages as Python lists, attention over gathered keys, drafts one by one."""
import math

import torch

E = 2.0 ** -24  # half a step of f32


def map_pages64(lens, add, tables, held, stack, page, capacity, max_tokens):
    """(status, tables, held, stack, slots, positions, starts, totals) from lists; nothing is
    moved where the step does not fit."""
    n, width = len(lens), len(tables[0])
    stay = (tables, held, stack, [-1] * max_tokens, [0] * max_tokens, [0] * (n + 1), list(lens))
    total = [a + b for a, b in zip(lens, add)]
    need = [-(-t // page) for t in total]
    back = sum(max(0, h - m) for h, m in zip(held, need))
    if (min(lens) < 0 or min(add) < 0 or max(total) > 2 ** 31 - 1 or max(need) > width or sum(add) > max_tokens or
            min(held) < 0 or max(held) > width):
        return (3,) + stay
    if sum(max(0, m - h) for h, m in zip(held, need)) > len(stack) + back:
        return (1,) + stay
    if len(stack) + back > capacity:
        return (3,) + stay
    tables, held, stack = [list(r) for r in tables], list(held), list(stack)
    for b in range(n):
        stack += tables[b][need[b]:held[b]]
    slots, positions, starts = [], [], [0]
    for b in range(n):
        for j in range(held[b], need[b]):
            tables[b][j] = stack.pop()
        held[b] = need[b]
        for p in range(lens[b], total[b]):
            positions.append(p)
            slots.append(tables[b][p // page] * page + p % page)
        starts.append(len(slots))
    behind = max_tokens - len(slots)
    return 0, tables, held, stack, slots + [-1] * behind, positions + [0] * behind, starts, total


def attend64(q, k_pages, v_pages, tables, lens, scale, starts, window, sinks, out):
    """(out, bound) in 64 bits: the formula, and what products and sums in f32 may be off by.

    A score's products and sums: head_dim products, each of parts that miss 2^-22 of it (4
    half steps) at most, and head_dim + 8 roundings of the running sum: (head_dim + 16) half
    steps of sum |q k| scale, and 2 of the score itself. A weight is off by that, twice (its
    own score's and the largest one's), and 8 half steps of exp2 and of its parts; the sums
    over keys are of 32 at a time, so keys / 32 + 64 roundings, in the numerator and in the
    denominator."""
    out = out.double()
    bound = torch.zeros_like(out)
    n_pages, page, kv, dim = k_pages.shape
    group = q.shape[1] // kv
    for b in range(tables.shape[0]):
        first, end = (b, b + 1) if starts is None else (int(starts[b]), int(starts[b + 1]))
        length = int(lens[b])
        if end == first:
            continue
        out[first:end], bound[first:end] = 0.0, 1e-30
        if length == 0:
            continue
        j = torch.arange(length, device=q.device)
        ids = tables[b].long()[j // page]
        real = (ids >= 0) & (ids < n_pages)
        rows = ids.clamp(0, n_pages - 1) * page + j % page
        p = length - (end - first) + torch.arange(end - first, device=q.device)[:, None]
        seen = (j <= p) & real
        if window:
            seen &= (j > p - window) | (j < sinks)
        some = seen.any(1)
        used = seen.any(0)
        for h in range(kv):
            k, v = (x.reshape(-1, kv, dim)[rows, h].double() for x in (k_pages, v_pages))
            k, v = (torch.where(used[:, None], x, 0.0) for x in (k, v))
            for g in range(group):
                x = q[first:end, h * group + g].double()
                raw = (x @ k.T) * scale
                s = raw.clamp(-100, 100).masked_fill(~seen, -math.inf)
                w = torch.softmax(torch.where(some[:, None], s, 0.0), -1)
                w = torch.where(seen, w, 0.0)
                y = torch.where(some[:, None], w @ v, 0.0)
                mag = (x.abs() @ k.abs().T) * abs(scale)
                ds = ((dim + 16) * mag + 2 * raw.abs()).masked_fill(~seen, 0.0).amax(1, keepdim=True)
                rel = 2 * ds + 8 + 2 * (length / 32 + 64)
                out[first:end, h * group + g] = y
                bound[first:end, h * group + g] = E * (rel * (w @ v.abs()) + 2 * y.abs()) + 1e-30
    return out, bound


def verify64(target, drafts, u, draft, counts):
    """(tokens, accepted) draft by draft, sums in 64 bits."""
    n, rows, vocab = target.shape
    k = rows - 1
    target, u = target.double().cpu(), u.double().cpu()
    draft = None if draft is None else draft.double().cpu()
    tokens, accepted = [], []
    for b in range(n):
        count = k if counts is None else min(max(int(counts[b]), 0), k)
        x = drafts[b].tolist()
        a = 0
        while a < count and 0 <= x[a] < vocab:
            q = 1.0 if draft is None else draft[b, a, x[a]].item()
            if not u[b, a].item() * q < target[b, a, x[a]].item():
                break
            a += 1
        plain = target[b, a]
        rest = plain.clone()
        if a < count:
            if draft is not None:
                rest = plain - draft[b, a]
            elif 0 <= x[a] < vocab:
                rest[x[a]] -= 1.0
        weigh = lambda r: torch.where(r > 0, r, 0.0)  # noqa: E731  (NaN weighs nothing)
        rest, plain = weigh(rest), weigh(plain)
        row = rest if (rest > 0).any() else plain
        run = torch.cumsum(row, 0)
        over = ((run > u[b, k] * run[-1]) & (row > 0)).nonzero()
        some = (row > 0).nonzero()
        token = int(over[0]) if len(over) else int(some[-1]) if len(some) else -1
        tokens.append(x[:a] + [token] + [-1] * (k - a))
        accepted.append(a)
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(accepted, dtype=torch.int32)
