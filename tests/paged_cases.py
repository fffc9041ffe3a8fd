"""Plain statements of the operators of a batch of requests of different lengths, in whole numbers and 64 bits, for the tests."""
import torch


def plan(cached, new, table, free, n_free, page, max_rows, pitch=0):
    """One request after another, as lists. Returns (lengths, n_free, starts, slots, positions, status), table and free changed in place."""
    B, width, n_pages = len(cached), len(table[0]) if table else 0, len(free)
    lengths, starts, status = list(cached), [], []
    slots, positions = [-1] * max_rows, [-1] * max_rows
    avail = max(0, min(n_free, n_pages))
    wanted, row, ended = 0, 0, []
    for b in range(B):
        n = max(new[b], 0)
        starts.append(b * pitch if pitch else row)
        row += n
        if cached[b] < 0 or cached[b] + n > width * page or (n and (starts[b] + n > max_rows or (pitch and n > pitch))):
            status.append(2)
            continue
        held = -(-cached[b] // page)
        if new[b] < 0:
            status.append(0)
            lengths[b] = 0
            ended.append((b, held))
            continue
        need = -(-(cached[b] + n) // page) - held
        wanted += need
        if need and wanted > avail:
            status.append(1)
            continue
        status.append(0)
        for j in range(need):
            table[b][held + j] = free[avail - 1 - (wanted - need) - j]
        lengths[b] = cached[b] + n
        for t in range(n):
            pos = cached[b] + t
            pg = table[b][pos // page]
            positions[starts[b] + t] = pos
            slots[starts[b] + t] = pg * page + pos % page if 0 <= pg < n_pages else -1
    starts.append(B * pitch if pitch else row)
    # a request that came too late for the free pages leaves no gap in what is taken: all behind it that need one are refused too
    taken = sum(-(-lengths[b] // page) + cached[b] // -page for b in range(B) if status[b] == 0 and new[b] >= 0)
    left = avail - taken
    for b, held in ended:
        for j in range(held):
            if left < n_pages:
                free[left] = table[b][j]
                left += 1
    return lengths, left, starts, slots, positions, status


def attention(q, k_pages, v_pages, table, lengths, hq, hk, d, scale=None):
    """(result in 64 bits, largest error that the kernel's arithmetic allows ahead of its last rounding), both [B, hq * d].
    Scores are sums of d exact products in 32 bits: |error| <= (d + 4) 2^-23 sum |q k|, and so is the weights' relative error (with one more of 2^-22 from the exponential); a weight enters
    as two bf16 terms: 2^-16 more. Numerator and denominator have it, and sums of n weights 2^-22 each."""
    B, G = q.shape[0], hq // hk
    scale = d ** -0.5 if scale is None else scale
    out, err = (torch.zeros(B, hq * d, dtype=torch.float64, device=q.device) for _ in range(2))
    page = k_pages.shape[1]
    for b, n in enumerate(lengths.tolist()):
        n = min(n, table.shape[1] * page)
        if n <= 0:
            continue
        ids = table[b, : -(-n // page)].long()
        ok = ((ids >= 0) & (ids < k_pages.shape[0])).repeat_interleave(page)[:n]
        ids = ids.clamp(0, k_pages.shape[0] - 1)
        k, v = (t[ids].reshape(-1, hk, d)[:n][ok].double().transpose(0, 1) for t in (k_pages, v_pages))
        if k.shape[1] == 0:
            out[b] = float("nan")
            continue
        qb = q[b].double().view(hk, G, d)
        s = qb @ k.transpose(1, 2) * scale
        w = torch.softmax(s, -1)
        size = (qb.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * abs(scale)
        rel = 2 * ((d + 4) * 2.0 ** -23 * size + 2.0 ** -16 + 2.0 ** -22) + n * 2.0 ** -22
        out[b] = (w @ v).reshape(-1)
        err[b] = (rel * (w @ v.abs())).reshape(-1)
    return out, err


def adjust(logits, tokens=None, lengths=None, prompt=None, rep=1.0, pres=0.0, freq=0.0, bias_ids=None, bias=None, mask=None):
    """(result in 64 bits, sum of the sizes of what was added up): every operation in 32 bits is off by 2^-24 of that at most."""
    x = logits.double().cpu().clone()
    B, V = x.shape
    size = x.abs()
    row_of = lambda v, b: float(v[b]) if isinstance(v, torch.Tensor) else float(v)
    for b in range(B):
        r, p, f = (float(torch.tensor(row_of(v, b), dtype=torch.float32)) for v in (rep, pres, freq))
        n = 0 if tokens is None else min(max(int(lengths[b]), 0), tokens.shape[1])
        words = tokens[b, :n].cpu() if n else torch.zeros(0, dtype=torch.int64)
        inside = (words >= 0) & (words < V)
        first = 0 if prompt is None else max(int(prompt[b]), 0)
        said = torch.bincount(words[inside], minlength=V)
        own = torch.bincount(words[first:][inside[first:]], minlength=V)
        hit = said > 0
        x[b][hit] = torch.where(x[b][hit] > 0, x[b][hit] / r, x[b][hit] * r)
        size[b] = size[b] + x[b].abs()
        x[b] -= f * own + p * (own > 0)
        size[b] += 2 * (abs(f) * own + abs(p) * (own > 0))
        if bias is not None:
            ids, vals = bias_ids[b].cpu(), bias[b].double().cpu()
            good = (ids >= 0) & (ids < V)
            x[b].index_add_(0, ids[good], vals[good])
            size[b].index_add_(0, ids[good], vals[good].abs() * ids.numel())
        if mask is not None:
            m = mask[b if mask.shape[0] > 1 else 0].cpu().long()
            bits = ((m[:, None] >> torch.arange(32)) & 1).view(-1)[:V]
            x[b][bits == 0] = float("-inf")
    return x, size
