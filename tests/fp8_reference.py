"""The operators of an FP8 expert layer written out in 64 bits with torch, as their definitions in the header say them."""
import math

import torch

BLOCK = 128
FP8_MAX = 448.0
AMAX_FLOOR = 2.0 ** -96


def blocks(n):
    return (n + BLOCK - 1) // BLOCK


def pad16(n):
    return (n + 15) // 16 * 16


def route(logits, bias, top_k, score, n_groups=1, top_groups=1, group_top=1, renorm=True, scale=1.0):
    """Row by row on the CPU; logits [rows, E], bias [E] or None -> idx int32, w float64."""
    x = logits.double().cpu()
    rows, experts = x.shape
    b = torch.zeros(experts, dtype=torch.float64) if bias is None else bias.double().cpu()
    idx, w = torch.full((rows, top_k), -1, dtype=torch.int32), torch.zeros(rows, top_k, dtype=torch.float64)
    for t in range(rows):
        row = x[t].clamp(max=torch.finfo(torch.float32).max)
        on = row > -math.inf                       # false for NaN
        if not on.any():
            continue
        if score == "sigmoid":
            s = torch.sigmoid(row)
        else:
            e = torch.exp(row - row[on].max())
            s = e / e[on].sum()
        s = torch.where(on, s, torch.zeros(()).double())
        p = torch.where(on & (b > -math.inf), s + b, torch.full((), -math.inf).double())
        p = torch.nan_to_num(p, nan=-math.inf, neginf=-math.inf, posinf=math.inf)
        if n_groups > 1:
            g = p.view(n_groups, -1)
            best = g.sort(dim=1, descending=True).values[:, :group_top]
            worth = torch.where(best[:, 0] > -math.inf, torch.where(best > -math.inf, best, 0.0).sum(1), -math.inf)
            stays = worth.sort(descending=True, stable=True).indices[:top_groups]
            keep = torch.zeros(n_groups, dtype=torch.bool)
            keep[stays] = True
            p = torch.where(keep[:, None], g, -math.inf).reshape(-1)
        value, order = p.sort(descending=True, stable=True)
        found = [int(e) for v, e in zip(value[:top_k], order[:top_k]) if v > -math.inf]
        picked = s[found]
        if renorm and len(found):
            picked = picked / picked.sum() if picked.sum() > 0 else picked * 0
        idx[t, :len(found)] = torch.tensor(found, dtype=torch.int32)
        w[t, :len(found)] = picked * scale
    return idx, w


def group(idx, experts):
    """Stable counting sort -> offsets, pair_row, row_pair (int32, CPU)."""
    flat = idx.cpu().view(-1).tolist()
    by_expert = [[] for _ in range(experts)]
    for p, e in enumerate(flat):
        if 0 <= e < experts:
            by_expert[e].append(p)
    offsets, row_pair = [0], []
    for pairs in by_expert:
        row_pair += pairs
        offsets.append(len(row_pair))
    pair_row = [-1] * len(flat)
    for r, p in enumerate(row_pair):
        pair_row[p] = r
    row_pair += [-1] * (len(flat) - len(row_pair))
    t = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return t(offsets), t(pair_row).view(idx.shape), t(row_pair)


def activation(x, act, limit=7.0, alpha=1.702):
    x = x.double()
    if act == "none":
        return x
    if act == "swiglu":
        gate, up = x[:, 0::2].clamp(max=limit), x[:, 1::2].clamp(-limit, limit)
        return gate * torch.sigmoid(alpha * gate) * (up + 1)
    half = x.shape[1] // 2
    return x[:, :half] * torch.sigmoid(x[:, :half]) * x[:, half:]


def quotient(a, b):
    """a / b rounded once to fp32 (the quotient of two fp32 values, rounded to 64 bits first, rounds to the same).  torch divides
    by a number, and a number by a tensor, through a rounded reciprocal."""
    return (torch.as_tensor(a, dtype=torch.float64) / torch.as_tensor(b, dtype=torch.float64)).float()


def quantise_rows(v):
    """fp32 [rows, cols] -> codes (float8) and scales, the definition's operations one by one in 32 bits."""
    rows, cols = v.shape
    b = torch.nn.functional.pad(v.float(), (0, blocks(cols) * BLOCK - cols)).view(rows, -1, BLOCK)
    a = b.abs()
    amax = torch.where(a < math.inf, a, 0.0).amax(2).clamp_min(AMAX_FLOOR)
    q = b * quotient(FP8_MAX, amax)[:, :, None]
    codes = q.clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).view(rows, -1)[:, :cols].contiguous()
    return codes, quotient(amax, FP8_MAX)


def quantise_blocks(w):
    """fp32 [mats, rows, cols] -> codes (float8) and scales [mats, row blocks, column blocks]."""
    mats, rows, cols = w.shape
    nb, kb = blocks(rows), blocks(cols)
    p = torch.zeros(mats, nb * BLOCK, kb * BLOCK, device=w.device)
    p[:, :rows, :cols] = w.float()
    p = p.view(mats, nb, BLOCK, kb, BLOCK)
    amax = p.abs().amax((2, 4)).clamp_min(AMAX_FLOOR)
    q = p * quotient(FP8_MAX, amax)[:, :, None, :, None]
    codes = q.clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn).view(mats, nb * BLOCK, kb * BLOCK)[:, :rows, :cols].contiguous()
    return codes, quotient(amax, FP8_MAX)


def gemm(a, sa, b, sb, offsets=None, bias=None):
    """a float8 [rows, k], b float8 [groups, n, k] -> the result in 64 bits, and the sum of the magnitudes of its terms."""
    rows, k = a.shape
    groups, n, _ = b.shape
    kk = torch.arange(k, device=a.device) // BLOCK
    nn = torch.arange(n, device=a.device) // BLOCK
    x = a.double() * sa.double()[:, kk]
    out = torch.zeros(rows, n, dtype=torch.float64, device=a.device)
    mag = torch.zeros_like(out)
    ends = [0, rows] if offsets is None else offsets.tolist()
    for g in range(groups):
        part = slice(ends[g], ends[g + 1])
        if ends[g + 1] <= ends[g]:
            continue
        w = b[g].double() * sb[g].double()[nn][:, kk]
        out[part], mag[part] = x[part] @ w.t(), x[part].abs() @ w.abs().t()
        if bias is not None:
            out[part] += bias[g].double()
            mag[part] += bias[g].double().abs()
    return out, mag


def combine(y, pair_row, w, residual=None):
    r = pair_row.long()
    on = (r >= 0) & (r < len(y))
    terms = torch.where(on[:, :, None], y.double()[r.clamp(0, max(0, len(y) - 1))] * w.double()[:, :, None], 0.0)
    out, mag = terms.sum(1), terms.abs().sum(1)
    if residual is not None:
        out, mag = out + residual.double(), mag + residual.double().abs()
    return out, mag
