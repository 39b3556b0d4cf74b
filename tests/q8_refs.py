"""The 8-bit cache in 64 bits: what ``store_q8``, ``paged_attention_q8`` and ``step_tables`` do, from their definitions, one token and one key at a time."""
import math

import torch

E4M3 = torch.float8_e4m3fn
F64 = torch.float64


def scale_of(most: float) -> float:
    """The least power of two s with most <= 448 s, between 2^-100 and 2^119."""
    e = -100
    while e < 119 and most > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def rounded(x):
    """float64 -> the nearest e4m3 number (ties to even), in float64: 3 bits behind the leading one, steps of 2^-9 below 2^-6, at most 448."""
    x = x.clamp(-448.0, 448.0)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    e = e + (x.abs() >= torch.exp2(e + 1)).to(F64) - (x.abs() < torch.exp2(e)).to(F64)      # a logarithm may be off in its last place
    step = torch.exp2(e.clamp(min=-6) - 3)
    return torch.where(x.isnan(), x, torch.round(x / step) * step)


def store(x, slots, cache, scale):
    """x [T, nkv, width] float64; cache [pages, nkv, page, width] and scale [pages, nkv], float64, updated in place."""
    ps = cache.shape[2]
    t, T = 0, len(slots)
    while t < T:
        s = int(slots[t])
        if s < 0 or s >= cache.shape[0] * ps:
            t += 1
            continue
        page, off, n = s // ps, s % ps, 1
        while t + n < T and int(slots[t + n]) == s + n and off + n < ps:
            n += 1
        for h in range(cache.shape[1]):
            part = x[t: t + n, h]
            fine = part[part.isfinite()]
            new = scale_of(float(fine.abs().max()) if fine.numel() else 0.0)
            old = float(scale[page, h])
            now = max(old, new) if off else new
            if off and now != old:
                cache[page, h, :off] = rounded(cache[page, h, :off] * (old / now))
            cache[page, h, off: off + n] = rounded(part / now)
            scale[page, h] = now
        t += n


def attention(q, k, v, ks, vs, indptr, kv_lens, table, nq, nkv, scale, window, sinks):
    """Returns (out, sum p |v|, largest |score|) in float64; q [T, nq * hd], caches as values of their codes."""
    hd, vd, ps = k.shape[3], v.shape[3], k.shape[2]
    T = q.shape[0]
    out, size = torch.zeros(T, nq * vd, dtype=F64, device=q.device), torch.zeros(T, nq * vd, dtype=F64, device=q.device)
    big = 0.0
    for r, kv in enumerate(kv_lens):
        for t in range(indptr[r], indptr[r + 1]):
            p = kv - (indptr[r + 1] - t)
            lo = max(0, p - window + 1) if window else 0
            if p < lo:
                continue
            j = torch.arange(lo, p + 1, device=q.device)
            page = table[r].to(q.device)[j // ps].long()
            kk = (k[page, :, j % ps].to(F64) * ks[page].to(F64)[:, :, None]).repeat_interleave(nq // nkv, dim=1)
            vv = (v[page, :, j % ps].to(F64) * vs[page].to(F64)[:, :, None]).repeat_interleave(nq // nkv, dim=1)
            s = torch.einsum("nhd,hd->hn", kk, q[t].to(F64).view(nq, hd)) * scale
            big = max(big, float(s.abs().nan_to_num(0.0, 0.0, 0.0).max()))
            m = s.amax(dim=1)
            if sinks is not None:
                m = torch.maximum(m, sinks.to(F64))
            w = torch.exp(s - m[:, None])
            total = w.sum(dim=1)
            if sinks is not None:
                total = total + torch.exp(sinks.to(F64) - m)
            w = w / total[:, None]
            out[t] = torch.einsum("hn,nhd->hd", w, vv).reshape(-1)
            size[t] = torch.einsum("hn,nhd->hd", w, vv.abs()).reshape(-1)
    return out, size, big


def tables(slots, starts, lens, new_pages, table, ps, width):
    """Lists of whole numbers; ``table`` (a list of lists) is updated."""
    indptr, kv, pos, row, sl, place, blocks = [0], [], [], [], [], [], []
    at = 0
    for r, (s, a, n) in enumerate(zip(slots, starts, lens)):
        for j in range(math.ceil(a / ps), math.ceil((a + n) / ps)):
            table[s][j] = new_pages[at]
            at += 1
        indptr.append(indptr[-1] + n)
        kv.append(a + n)
        have = math.ceil((a + n) / ps)
        blocks.append([table[s][j] if j < have else -1 for j in range(width)])
        for p in range(a, a + n):
            pos.append(p), row.append(r), sl.append(s), place.append(table[s][p // ps] * ps + p % ps)
    return indptr, kv, pos, row, sl, place, blocks
