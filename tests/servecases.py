"""Plain 64-bit forms of the batch serving operators, and calls of the
library's own, for the tests (numpy on the host, torch only to hold device
memory)."""
import ctypes as C

import numpy as np
import torch

import kmap_b200 as K

DEV = "cuda"
FORMATS = {"f32": K.KV_F32, "i8": K.KV_I8, "e4m3": K.KV_E4M3}
QMAX = {"i8": np.float32(127), "e4m3": np.float32(448)}
#: the 127 magnitudes of an e4m3 code, in code order
E4M3 = np.array([(m / 8 * 2.0 ** -6) if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                 for e in range(16) for m in range(8)][:127])


def rope32(x, cos, sin):
    """Rotate-half in the tape's fp32 arithmetic; x [rows][heads][hd], cos / sin [rows][hd]."""
    h = x.shape[-1] // 2
    o = np.concatenate([-x[..., h:], x[..., :h]], -1)
    return x * cos[:, None] + o * sin[:, None]


def quantise(x, fmt):
    """(codes as numbers, scales) of fp32 rows x[..., hd], by the definition in fp32."""
    if fmt == "f32":
        return x, None
    x = np.asarray(x, np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        amax = np.maximum(np.abs(x).max(-1), np.float32(2.0 ** -100))
        y = (x * (QMAX[fmt] / amax)[..., None]).astype(np.float64)
        most = np.float32(np.finfo(np.float32).max / float(QMAX[fmt]))
        if float(most) * float(QMAX[fmt]) > np.finfo(np.float32).max:
            most = np.nextafter(most, np.float32(0))
        scale = np.minimum(amax / QMAX[fmt], most)
    if fmt == "i8":
        codes = np.rint(y)
    else:
        # the nearest magnitude, ties to the even code
        a = np.minimum(np.abs(np.nan_to_num(y)), 448.0)
        hi = np.searchsorted(E4M3, a).clip(1, 126)
        lo = hi - 1
        dl, dh = a - E4M3[lo], E4M3[hi] - a
        c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
        codes = np.copysign(E4M3[c], y)
    bad = ~np.isfinite(x).all(-1)
    codes = np.where(bad[..., None], 0.0, codes)
    return codes, np.where(bad, np.float32(np.nan), scale).astype(np.float32)


def values32(codes, scale):
    return np.float32(codes) if scale is None else np.float32(codes) * scale[..., None]


class Cache:
    """A device cache with `pad` spare elements between sequences."""

    def __init__(self, fmt, n_seq, n_kv, max_pos, hd, pad=0, fill=0):
        self.fmt, self.hd, self.n_seq, self.n_kv, self.max_pos = fmt, hd, n_seq, n_kv, max_pos
        self.stride, self.sstride = n_kv * max_pos * hd + pad, n_kv * max_pos + pad
        kind = torch.float32 if fmt == "f32" else torch.uint8
        self.k = torch.full((n_seq, self.stride), fill, dtype=kind, device=DEV)
        self.v = torch.full((n_seq, self.stride), fill, dtype=kind, device=DEV)
        self.ks = torch.full((n_seq, self.sstride), float("nan"), device=DEV)
        self.vs = torch.full((n_seq, self.sstride), float("nan"), device=DEV)
        self.c = K.KvCache(FORMATS[fmt], n_seq, n_kv, hd, max_pos, self.k.data_ptr(),
                           self.v.data_ptr(), self.ks.data_ptr(), self.vs.data_ptr(), self.stride,
                           self.sstride)

    def by(self):
        return C.byref(self.c)

    def raw(self, name):
        """Codes as numbers [seq][kv][pos][hd] and scales [seq][kv][pos]."""
        t = getattr(self, name)[:, :self.n_kv * self.max_pos * self.hd].cpu()
        if self.fmt == "i8":
            t = t.view(torch.int8)
        elif self.fmt == "e4m3":
            t = t.view(torch.float8_e4m3fn).float()
        shape = (self.n_seq, self.n_kv, self.max_pos, self.hd)
        s = getattr(self, name + "s")[:, :self.n_kv * self.max_pos].cpu().numpy().reshape(shape[:3])
        return t.numpy().astype(np.float64).reshape(shape), None if self.fmt == "f32" else s

    def put(self, name, x):
        """Store fp32 rows x [seq][kv][n][hd] at positions 0..n-1, by the plain definition."""
        codes, scale = quantise(x, self.fmt)
        n = x.shape[2]
        t = torch.from_numpy(np.float32(codes))
        if self.fmt == "i8":
            t = t.to(torch.int8).view(torch.uint8)
        elif self.fmt == "e4m3":
            t = t.to(torch.float8_e4m3fn).view(torch.uint8)
        full = self.n_kv * self.max_pos
        view = getattr(self, name)[:, :full * self.hd].view(self.n_seq, self.n_kv, self.max_pos, self.hd)
        view[:, :, :n] = t.to(DEV)
        if scale is not None:
            view = getattr(self, name + "s")[:, :full].view(self.n_seq, self.n_kv, self.max_pos)
            view[:, :, :n] = torch.from_numpy(scale).to(DEV)
        return values32(codes, scale).astype(np.float64)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEV)


def attend(q, k, v, scale):
    """Attention of rows q [G][hd] over k, v [n][hd], 64 bits; zeros without positions.
    Returns the output and an error bound's two ingredients per row:
    max over positions of sum |q k| * scale, and max |v|."""
    if len(k) == 0:
        return np.zeros_like(q), np.zeros(len(q)), 0.0
    s = q @ k.T * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    return p @ v / p.sum(-1, keepdims=True), (np.abs(q) @ np.abs(k).T * scale).max(-1), np.abs(v).max()


def run_attention(q, out, n_heads, scale, prefix=None, prefix_len=0, own=None, lens=None,
                  max_len=0, stream=None):
    """kllm_batch_attention on device tensors q, out [n_seq][stride]."""
    n = q.shape[0]
    a = K.BatchAttn(n, n_heads, prefix_len, max_len, scale, q.data_ptr(), q.stride(0),
                    C.addressof(prefix.c) if prefix else None,
                    C.addressof(own.c) if own else None,
                    lens.data_ptr() if lens is not None else None, out.data_ptr(), out.stride(0),
                    None, 0)
    size = K.lib().kllm_batch_attention_workspace(C.byref(a))
    assert size > 0, K.last_error()
    # what lies behind the workspace has to stay as it is
    ws = torch.full((size + 64,), 0xa5, dtype=torch.uint8, device=DEV)
    a.workspace, a.workspace_bytes = ws.data_ptr(), size
    K.check(K.lib().kllm_batch_attention(C.byref(a), stream), "kllm_batch_attention")
    torch.cuda.synchronize()
    assert bool((ws[size:] == 0xa5).all())
    return ws


def sample_plain(x, T, k, p, mp, u):
    """The token of one row of logits (fp32), by the definition in 64 bits."""
    x = np.asarray(x, np.float64)
    nan0 = np.isnan(x[0])
    x = np.where(np.isnan(x), -np.inf, x)
    if T <= 0:
        return 0 if nan0 else int(x.argmax())
    top = x.max()
    if top == -np.inf:
        return 0
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / T))
    w = np.nan_to_num(w)
    order = np.argsort(-x, kind="stable")
    n = len(x) if k <= 0 else min(k, len(x))
    mass = np.concatenate([[0.0], np.cumsum(w[order[:n]])])
    if p < 1:
        n = max(1, int((mass[:n] < p * mass[n]).sum()))
    if mp > 0:
        while n > 1 and w[order[n - 1]] < min(mp, 1.0):
            n -= 1
    kept = np.sort(order[:n])
    c = np.cumsum(w[kept])
    u = u if u > 0 else 0.0
    u = min(u, 1 - 2.0 ** -24)
    return int(kept[min(int((c <= u * c[-1]).sum()), n - 1)])


def sample_args(x, T=None, k=None, p=None, mp=None, u=None, vocab=None):
    """kllm_sample's arguments for rows x (device tensor [rows][stride]), the
    tokens (one more than there are) and what they point to."""
    rows = x.shape[0]
    t = [None if a is None else dev(np.asarray(a, d)) for a, d in
         ((T, np.float32), (k, np.int32), (p, np.float32), (mp, np.float32), (u, np.float32))]
    out = torch.full((rows + 1,), -7, dtype=torch.int32, device=DEV)
    ptr = [None if a is None else a.data_ptr() for a in t]
    return K.SampleRows(rows, vocab or x.shape[1], x.data_ptr(), x.stride(0), *ptr, out.data_ptr()), out, t


def run_sample(x, *settings, vocab=None, stream=None, **named):
    a, out, _keep = sample_args(x, *settings, vocab=vocab, **named)
    K.check(K.lib().kllm_sample(C.byref(a), stream), "kllm_sample")
    torch.cuda.synchronize()
    assert int(out[-1]) == -7
    return out[:-1].cpu().numpy()
