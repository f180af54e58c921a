"""What is measured of the batch-serving operators, and their plain forms.

Three operators: the key/value cache that is quantised as it is written and
read back (op "kv"), the decode attention of a batch that shares a prefix (op
"attn"), and the draw of tokens from logits (op "sample").  `run` computes
them from elementary torch operations, or with `own` set through the
library's entry points."""
import ctypes
import math

import numpy as np
import torch

own = False

#: heads, kv heads, head dim, positions: the TinyLlama, 7B and 8B
#: architectures of the chip generator
ARCH = {"1b": (32, 4, 64, 2048), "7b": (32, 32, 128, 4352), "8b": (32, 8, 128, 1152)}
FORMATS = ("f32", "i8", "e4m3")
QMAX = {"i8": 127.0, "e4m3": 448.0}
TINY = 2.0 ** -100


# ------------------------------------------------------------------ cases --

def _kv(name, arch, fmt, rows, prompt):
    return {"name": name, "op": "kv", "arch": arch, "fmt": fmt, "rows": rows, "prompt": prompt}


def _attn(name, arch, fmt, seqs, prefix, own_len):
    return {"name": name, "op": "attn", "arch": arch, "fmt": fmt, "seqs": seqs, "prefix": prefix,
            "own_len": own_len}


def _sample(name, rows, vocab, mode, ties=False):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "mode": mode, "ties": ties}


def listed():
    return [
        # one sequence's step: latency
        _kv("kv-1b-i8-1row", "1b", "i8", 1, False),
        # a step of 32 sequences
        _kv("kv-8b-e4m3-32rows", "8b", "e4m3", 32, False),
        # a long prompt's positions written after its pass, read back for the next
        _kv("kv-7b-i8-prompt4095", "7b", "i8", 4095, True),
        # a few answers to a short prompt: latency
        _attn("attn-1b-i8-4x97", "1b", "i8", 4, 97, 33),
        # an odd batch on a middling prompt, eight heads per kv head of 64
        _attn("attn-1b-e4m3-33x2047", "1b", "e4m3", 33, 2047, 161),
        # 32 answers to a 1024-token prompt
        _attn("attn-8b-i8-32x1024", "8b", "i8", 32, 1024, 128),
        # the largest: 64 answers to a long document
        _attn("attn-8b-e4m3-64x16384", "8b", "e4m3", 64, 16384, 512),
        # fp32 caches, one query head per kv head
        _attn("attn-7b-f32-24x4000", "7b", "f32", 24, 4000, 300),
        # no prefix: ragged sequences of their own
        _attn("attn-8b-i8-48-ragged", "8b", "i8", 48, 0, 4352),
        # one sequence's draw, top-k and top-p
        _sample("sample-1x32000", 1, 32000, "mixed"),
        # a step of 32 sequences with settings of their own
        _sample("sample-32x128256", 32, 128256, "mixed"),
        # many rows, nucleus only, logits rounded to bf16 (many equal ones)
        _sample("sample-128x128256-ties", 128, 128256, "top_p", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["kv", "attn", "attn", "sample"])
    if op == "kv":
        arch = rng.choice(list(ARCH))
        prompt = rng.random() < 0.5
        rows = _log(rng, 1, ARCH[arch][3] - 1 if prompt else 128)
        return {"op": "kv", "arch": arch, "fmt": rng.choice(FORMATS), "rows": min(rows, 4095),
                "prompt": prompt}
    if op == "attn":
        arch, fmt = rng.choice(list(ARCH)), rng.choice(FORMATS)
        most = [work(c) for c in listed()]
        while True:
            c = {"op": "attn", "arch": arch, "fmt": fmt, "seqs": _log(rng, 1, 64),
                 "prefix": rng.choice([0, 1, 1, 1]) * _log(rng, 1, 16384),
                 "own_len": _log(rng, 1, 4352)}
            w = work(c)
            if all(w[k] <= max(m[k] for m in most) for k in w):
                return c
    return {"op": "sample", "rows": _log(rng, 1, 128), "vocab": _log(rng, 1000, 128256),
            "mode": rng.choice(["mixed", "top_p", "top_k", "min_p", "plain"]),
            "ties": rng.random() < 0.3}


# ----------------------------------------------------------------- inputs --

def _lens(n, most):
    """How many positions of its own each of n sequences has: 1 to `most`, spread evenly."""
    return [1 + (most - 1) * i // max(n - 1, 1) if n > 1 else most for i in range(n)]


def _quantise(x, fmt):
    """Codes and scales of rows x[..., hd] (fp32)."""
    if fmt == "f32":
        return x, None
    amax = x.abs().amax(-1).clamp(min=TINY)
    q = torch.full_like(amax, QMAX[fmt])     # tensors on both sides: a division rounded once
    y = x * (q / amax).unsqueeze(-1)
    codes = torch.round(y).to(torch.int8) if fmt == "i8" else y.to(torch.float8_e4m3fn)
    return codes, amax / q


def _values(codes, scale):
    return codes if scale is None else codes.float() * scale.unsqueeze(-1)


def _cache(g, seqs, nkv, positions, hd, fmt, dev):
    """A filled cache: codes [seq][kv head][position][hd] and scales, of k and of v."""
    c = {}
    for name in "kv":
        x = torch.randn(seqs, nkv, positions, hd, generator=g, device=dev)
        x *= 0.5 + torch.rand(seqs, nkv, positions, 1, generator=g, device=dev)
        c[name], c[name + "s"] = _quantise(x, fmt)
        del x
    return c


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "sample":
        rows, V = case["rows"], case["vocab"]
        # a bulk of unlikely tokens and a few tens that stand out
        x = torch.randn(rows, V, generator=g, device=dev) * 1.5
        hot = torch.randint(0, V, (rows, 40), generator=g, device=dev)
        x.scatter_add_(1, hot, 9 * torch.rand(rows, 40, generator=g, device=dev))
        s["logits"] = x.bfloat16().float() if case["ties"] else x
        r = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=g, device=dev)
        off = torch.ones(rows, device=dev)
        which = torch.arange(rows, device=dev) % 4
        mode = case["mode"]
        s["temperature"] = r(0.6, 1.3)
        s["top_p"] = r(0.7, 0.98) if mode in ("mixed", "top_p") else off
        s["top_k"] = torch.randint(1, 200, (rows,), generator=g, device=dev, dtype=torch.int32)
        if mode not in ("mixed", "top_k"):
            s["top_k"].zero_()
        s["min_p"] = r(0.001, 0.1) if mode in ("mixed", "min_p") else 0 * off
        if mode == "mixed":   # a greedy row, rows without a top-k, rows without a top-p
            s["temperature"][which == 3] = 0
            s["top_k"][which == 1] = 0
            s["top_p"][which == 2] = 1
        s["u"] = torch.rand(rows, generator=g, device=dev)
        return s
    nh, nkv, hd, mp = ARCH[case["arch"]]
    if case["op"] == "kv":
        rows, fmt = case["rows"], case["fmt"]
        seqs = 1 if case["prompt"] else rows
        s["qkv"] = torch.randn(rows, (nh + 2 * nkv) * hd, generator=g, device=dev)
        inv = 10000.0 ** (-torch.arange(0, hd, 2, device=dev, dtype=torch.float64) / hd)
        a = torch.arange(mp, device=dev, dtype=torch.float64)[:, None] * torch.cat([inv, inv])
        s["cos"], s["sin"] = a.cos().float(), a.sin().float()
        s["pos0"] = 0
        if not case["prompt"]:
            s["pos"] = torch.randint(0, mp, (rows,), generator=g, device=dev, dtype=torch.int32)
        kind = {"f32": torch.float32, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}[fmt]
        for name in "kv":
            s[name] = torch.zeros(seqs, nkv, mp, hd, device=dev, dtype=torch.float32).to(kind)
            s[name + "s"] = None if fmt == "f32" else torch.zeros(seqs, nkv, mp, device=dev)
        return s
    n = case["seqs"]
    # queries long enough that a few positions stand out
    s["q"] = 2 * torch.randn(n, nh * hd, generator=g, device=dev)
    s["prefix"] = _cache(g, 1, nkv, case["prefix"], hd, case["fmt"], dev) if case["prefix"] else None
    s["own"] = _cache(g, n, nkv, case["own_len"], hd, case["fmt"], dev)
    lens = torch.tensor(_lens(n, case["own_len"]), dtype=torch.int32, device=dev)
    s["lens"] = lens[torch.randperm(n, generator=g, device=dev)].contiguous()
    return s


# ------------------------------------------------------------ plain forms --

def _rope(x, cos, sin):
    h = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., h:], x[..., :h]], -1) * sin


def _kv_plain(s):
    case = s["case"]
    nh, nkv, hd, mp = ARCH[case["arch"]]
    rows = case["rows"]
    x = s["qkv"].view(rows, nh + 2 * nkv, hd)
    if case["prompt"]:
        seq = torch.zeros(rows, dtype=torch.long, device=x.device)
        pos = s["pos0"] + torch.arange(rows, device=x.device)
    else:
        seq, pos = torch.arange(rows, device=x.device), s["pos"].long()
    y = _rope(x[:, :nh + nkv], s["cos"][pos][:, None], s["sin"][pos][:, None])
    out = [y[:, :nh].reshape(rows, nh * hd)]
    for name, new in (("k", y[:, nh:]), ("v", x[:, nh + nkv:])):
        codes, scale = _quantise(new, case["fmt"])
        # byte-sized floats are moved as bytes
        cache = s[name].view(torch.uint8) if case["fmt"] == "e4m3" else s[name]
        cache[seq, :, pos] = codes.view(torch.uint8) if case["fmt"] == "e4m3" else codes
        if scale is not None:
            s[name + "s"][seq, :, pos] = scale
        got = cache[seq, :, pos]
        if case["fmt"] == "e4m3":
            got = got.view(torch.float8_e4m3fn)
        out.append(_values(got, None if scale is None else s[name + "s"][seq, :, pos]))
    return out


def _attn_plain(s):
    case = s["case"]
    nh, nkv, hd, _ = ARCH[case["arch"]]
    n, G, scale = case["seqs"], nh // nkv, 1 / math.sqrt(hd)
    q = s["q"].view(n, nkv, G, hd)
    o = s["own"]
    k, v = _values(o["k"], o["ks"]), _values(o["v"], o["vs"])
    sc = torch.matmul(q, k.transpose(2, 3)) * scale                       # [n][nkv][G][own]
    gone = torch.arange(k.shape[2], device=q.device) >= s["lens"][:, None]
    sc = torch.where(gone[:, None, None], -math.inf, sc)
    m = sc.amax(-1, keepdim=True)
    if s["prefix"]:
        p = s["prefix"]
        pk, pv = _values(p["k"], p["ks"])[0], _values(p["v"], p["vs"])[0]
        ps = torch.matmul(q.permute(1, 0, 2, 3).reshape(nkv, n * G, hd), pk.transpose(1, 2)) * scale
        pm = ps.amax(-1).view(nkv, n, G, 1).permute(1, 0, 2, 3)
        m = torch.maximum(m, pm)
        pe = torch.exp(ps - m.permute(1, 0, 2, 3).reshape(nkv, n * G, 1))
    e = torch.exp(sc - m)
    l, out = e.sum(-1, keepdim=True), torch.matmul(e, v)
    if s["prefix"]:
        l = l + pe.sum(-1).view(nkv, n, G, 1).permute(1, 0, 2, 3)
        out = out + torch.matmul(pe, pv).view(nkv, n, G, hd).permute(1, 0, 2, 3)
    return (out / l).reshape(n, nh * hd)


def _sample_plain(s):
    x = s["logits"]
    rows, V = x.shape
    xs, order = torch.sort(x, dim=-1, descending=True, stable=True)       # ties: the lowest index first
    T = s["temperature"].double()[:, None]
    greedy = T <= 0
    top = xs[:, :1].double()
    w = torch.exp((xs.double() - top) / torch.where(greedy, 1.0, T))
    rank = torch.arange(V, device=x.device)
    k = s["top_k"].long()[:, None]
    keep = (rank < k) | (k <= 0)
    cum = torch.cumsum(w * keep, -1)
    p = s["top_p"].double()[:, None]
    keep &= (cum - w < p * cum[:, -1:]) | (p >= 1) | (rank == 0)
    keep &= (w >= s["min_p"].double()[:, None]) | (rank == 0)
    keep &= ~greedy | (rank == 0)
    kept = torch.zeros_like(w).scatter_(1, order, w * keep)
    cum = torch.cumsum(kept, -1)
    return (cum <= s["u"].double()[:, None] * cum[:, -1:]).sum(-1).clamp(max=V - 1).int()


# -------------------------------------------------------- the framework's --

def _struct(K, c, fmt, hd):
    k, v, ks, vs = c["k"], c["v"], c["ks"], c["vs"]
    n, nkv, mp = k.shape[:3]
    return K.KvCache(FORMATS.index(fmt), n, nkv, hd, mp, k.data_ptr(), v.data_ptr(),
                     ks.data_ptr() if ks is not None else None,
                     vs.data_ptr() if vs is not None else None, nkv * mp * hd, nkv * mp)


def _run_own(s):
    import kmap_b200 as K
    case, stream = s["case"], torch.cuda.current_stream().cuda_stream
    lib, by = K.lib(), ctypes.byref
    if case["op"] == "sample":
        x = s["logits"]
        rows, V = x.shape
        out = torch.empty(rows, dtype=torch.int32, device=x.device)
        a = K.SampleRows(rows, V, x.data_ptr(), V, s["temperature"].data_ptr(), s["top_k"].data_ptr(),
                         s["top_p"].data_ptr(), s["min_p"].data_ptr(), s["u"].data_ptr(),
                         out.data_ptr())
        K.check(lib.kllm_sample(by(a), stream), "kllm_sample")
        return out
    nh, nkv, hd, mp = ARCH[case["arch"]]
    if case["op"] == "kv":
        rows, x = case["rows"], s["qkv"]
        cache = _struct(K, s, case["fmt"], hd)
        q = torch.empty(rows, nh * hd, device=x.device)
        k = torch.empty(rows, nkv, hd, device=x.device)
        v = torch.empty(rows, nkv, hd, device=x.device)
        at = x.data_ptr()
        pos = None if case["prompt"] else s["pos"].data_ptr()
        r = K.KvRows(rows, nh, s["pos0"], mp, 0, None, pos, at, at + 4 * nh * hd,
                     at + 4 * (nh + nkv) * hd, x.shape[1], hd, q.data_ptr(), s["cos"].data_ptr(),
                     s["sin"].data_ptr())
        K.check(lib.kllm_kv_append(by(cache), by(r), stream), "kllm_kv_append")
        K.check(lib.kllm_kv_read(by(cache), rows, None, pos, s["pos0"], k.data_ptr(), v.data_ptr(),
                                 nkv * hd, hd, stream), "kllm_kv_read")
        return [q, k, v]
    n, q = case["seqs"], s["q"]
    out = torch.empty_like(q)
    o = _struct(K, s["own"], case["fmt"], hd)
    p = _struct(K, s["prefix"], case["fmt"], hd) if s["prefix"] else None
    a = K.BatchAttn(n, nh, case["prefix"], case["own_len"], 1 / math.sqrt(hd), q.data_ptr(), nh * hd,
                    ctypes.addressof(p) if p else None, ctypes.addressof(o), s["lens"].data_ptr(),
                    out.data_ptr(), nh * hd, None, 0)
    if "workspace" not in s:   # kept from step to step, as its size is
        size = lib.kllm_batch_attention_workspace(by(a))
        s["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device=q.device)
    a.workspace, a.workspace_bytes = s["workspace"].data_ptr(), s["workspace"].numel()
    K.check(lib.kllm_batch_attention(by(a), stream), "kllm_batch_attention")
    return out


def run(state):
    if own:
        return _run_own(state)
    return {"kv": _kv_plain, "attn": _attn_plain, "sample": _sample_plain}[state["case"]["op"]](state)


# ------------------------------------------------------------------- work --

def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 24 * case["rows"], "flops": 4 * n}
    nh, nkv, hd, _ = ARCH[case["arch"]]
    per = 4 * hd if case["fmt"] == "f32" else hd + 4         # bytes of one position and head of k or v
    if case["op"] == "kv":
        new = 4 * (nh + 2 * nkv) * hd + 4 * nh * hd + 2 * nkv * per      # append
        back = 2 * nkv * per + 8 * nkv * hd                              # read back
        angles = 8 * hd * case["rows"]
        return {"bytes": case["rows"] * (new + back) + angles, "flops": 10 * case["rows"] * (nh + 2 * nkv) * hd}
    n, total = case["seqs"], sum(_lens(case["seqs"], case["own_len"]))
    return {"bytes": 2 * nkv * per * (case["prefix"] + total) + 8 * n * nh * hd,
            "flops": 4 * hd * nh * (n * case["prefix"] + total)}


# ------------------------------------------------- the definitions, 64 bits --

def _exact_rows(x, fmt):
    """Rows x (fp32 numpy) as the cache holds them.  Which code a value gets is defined by fp32
    arithmetic, rn(fl(x * fl(Q / amax))), as the tape's rotation is, so that every implementation
    stores the same codes; the value a code stands for is code * amax / Q."""
    if fmt == "f32":
        return x.astype(np.float64)
    amax = np.maximum(np.abs(x).max(-1, keepdims=True), np.float32(TINY))
    y = (x * (np.float32(QMAX[fmt]) / amax)).astype(np.float64)
    scale = amax.astype(np.float64) / QMAX[fmt]
    if fmt == "i8":
        return np.rint(y) * scale
    # e4m3: three fraction bits, exponents from -6
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
    return np.clip(np.rint(y / step) * step, -448, 448) * scale


def _exact_sample(s):
    x, out = s["logits"].cpu().numpy().astype(np.float64), []
    f = {n: s[n].cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p", "u")}
    for r in range(x.shape[0]):
        T = float(f["temperature"][r])
        if T <= 0:
            out.append(int(x[r].argmax()))
            continue
        w = np.exp((x[r] - x[r].max()) / T)
        order = np.argsort(-x[r], kind="stable")
        n = len(order) if f["top_k"][r] <= 0 else min(int(f["top_k"][r]), len(order))
        mass = np.concatenate([[0.0], np.cumsum(w[order[:n]])])
        if f["top_p"][r] < 1:
            n = max(1, int(np.searchsorted(mass[:n], float(f["top_p"][r]) * mass[n], side="left")))
        while n > 1 and w[order[n - 1]] < float(f["min_p"][r]):
            n -= 1
        kept = np.sort(order[:n])
        c = np.cumsum(w[kept])
        out.append(int(kept[min(int(np.searchsorted(c, float(f["u"][r]) * c[-1], side="right")), n - 1)]))
    return torch.tensor(out, dtype=torch.int32)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    nh, nkv, hd, _ = ARCH[case["arch"]]
    if case["op"] == "kv":
        rows, h = case["rows"], hd // 2
        x = s["qkv"].cpu().numpy().reshape(rows, nh + 2 * nkv, hd)
        pos = s["pos0"] + np.arange(rows) if case["prompt"] else s["pos"].cpu().numpy()
        c, d = (s[t].cpu().numpy()[pos][:, None] for t in ("cos", "sin"))

        def turn(x, c, d):
            a, b = x[..., :h], x[..., h:]
            return np.concatenate([a * c[..., :h] - b * d[..., :h], b * c[..., h:] + a * d[..., h:]], -1)

        q = turn(*(t.astype(np.float64) for t in (x[:, :nh], c, d)))
        return [torch.from_numpy(v) for v in (q.reshape(rows, nh * hd),
                                              _exact_rows(turn(x[:, nh:nh + nkv], c, d), case["fmt"]),
                                              _exact_rows(x[:, nh + nkv:], case["fmt"]))]
    n, G = case["seqs"], nh // nkv
    val = lambda c, name, i, h, e: (c[name][i, h, :e].double() if c[name + "s"] is None else
                                    c[name][i, h, :e].double() * c[name + "s"][i, h, :e, None].double())
    out = torch.empty(n, nkv, G, hd, dtype=torch.float64, device="cuda")
    q, lens = s["q"].double().view(n, nkv, G, hd), s["lens"].tolist()
    for h in range(nkv):
        pre = [val(s["prefix"], name, 0, h, case["prefix"]) for name in "kv"] if s["prefix"] else None
        for i in range(n):
            k, v = (val(s["own"], name, i, h, lens[i]) for name in "kv")
            if pre:
                k, v = torch.cat([pre[0], k]), torch.cat([pre[1], v])
            out[i, h] = torch.softmax(q[i, h] @ k.t() / math.sqrt(hd), -1) @ v
    return out.view(n, nh * hd)
