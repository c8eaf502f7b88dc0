"""The 8-bit cache and its attention in 64 bits, sequence by sequence, from the definition alone."""
import torch

EPS = 2.0 ** -23


def new_rows(qkv, cos, sin, p, h, d):
    """Rotated and normalised query and key, and the value, of one packed row; fp64 ``[H, D]`` each."""
    q, k, v = qkv.double().view(3, h, d).unbind(0)
    c, s = cos[p].double(), sin[p].double()
    out = []
    for x in (q, k):
        a, b = x[:, :d // 2], x[:, d // 2:]
        y = torch.cat([a * c + b * s, b * c - a * s], -1)
        out.append(y / (y.square().mean(-1, keepdim=True) + EPS).sqrt())
    return out[0], out[1], v


def held(cache, b, n):
    """What the cache holds of sequence b's first n tokens, fp64 ``[H, n, D]``: codes times scales, the open block as it is."""
    k8, v8, ks, vs, kt, vt = cache
    _, h, _, d = k8.shape
    full = n // 64
    nan = torch.full((), float("nan"), dtype=torch.float64, device=k8.device)
    kc = k8[b, :, :full * 64].view(h, full, 64, d)
    vc = v8[b, :, :full].transpose(-1, -2)
    k = torch.where(kc == -128, nan, kc.double() * ks[b, :, :full].double().abs()[..., None, None]).reshape(h, full * 64, d)
    v = torch.where(vc == -128, nan, vc.double() * vs[b, :, :full].double().abs()[..., None, None]).reshape(h, full * 64, d)
    rest = n - full * 64
    return torch.cat([k, kt[b, :, :rest].double()], 1), torch.cat([v, vt[b, :, :rest].double()], 1)


def first_key(p, start, window):
    return max(start, (p // 128 - (window // 128 - 1)) * 128 if window else 0, 0)


def attend(qkv, cos, sin, before, new_k, pos, scale, doc_start, window):
    """``y [B, H, D]`` in fp64 from the cache as it was before the step and the new keys ``new_k [B, H, D]`` as it keeps them (bf16),
    and the largest |v| that each sequence sees."""
    nseq, h, cap, d = before[0].shape
    y = torch.zeros(nseq, h, d, dtype=torch.float64, device=qkv.device)
    most = torch.zeros(nseq, dtype=torch.float64, device=qkv.device)
    for b, p in enumerate(pos):
        lo = first_key(p, int(doc_start[b]) if doc_start is not None else 0, window)
        if p < 0 or p >= min(cap, cos.shape[0]) or lo > p:
            continue
        q, _, v = new_rows(qkv[b], cos, sin, p, h, d)
        v = v.to(torch.bfloat16).double()                  # as the open block keeps it
        k_all, v_all = held(before, b, p)
        k_all, v_all = torch.cat([k_all, new_k[b].double()[:, None]], 1)[:, lo:], torch.cat([v_all, v[:, None]], 1)[:, lo:]
        w = torch.softmax(torch.einsum("hd,hnd->hn", q, k_all) * scale, -1)
        y[b] = torch.einsum("hn,hnd->hd", w, v_all)
        most[b] = v_all.abs().max()
    return y, most
