"""Paged-cache operators of serving, measured against their plain forms.

Four operators, each on the geometries this package's workloads use (32 query heads over 8 or 32 key/value heads of 128
channels, 6 heads of 48) and generic ones around them:

* ``append``   -- RMS norm of each query and key head, rotary positions (two pairings, part of the head, scaled for long
  contexts) and the append of keys and values to a paged cache, held in fp32 or in 4 bits;
* ``attend4``  -- attention over a paged cache held in 4 bits: one query row per sequence, or a ragged chunk of rows;
* ``index``    -- minimum and maximum of the keys of each cache block, brought up to date behind appended tokens;
* ``sparse``   -- decode attention over the blocks that this index scores highest for each sequence and key/value head.

The 4-bit cache holds a value as sign * {0, .5, 1, 1.5, 2, 3, 4, 6} * 2^e, one e for each 32 channels of a row: the
smallest with |row| <= 7 * 2^e; values are rounded to the nearest, ties to the even code.
"""
import math
import random

import torch

own = False

DEV = "cuda"
THETA = 10000.0
EPS = 1e-5
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of one request: what a single user waits for between two tokens
        dict(name="append_1_row", op="append", cache="fp32", rows=1, seqs=1, n_heads=32, n_kv=8, hd=128, bs=16, far=2048,
             layout="interleaved", rotary=128, scaling="none", norm=False),
        # a decode step of a full batch at far positions: normed heads, half pairing, a context stretched eight times
        dict(name="append_256_rows_4bit", op="append", cache="mx4", rows=256, seqs=256, n_heads=32, n_kv=8, hd=128, bs=16,
             far=32768, layout="half", rotary=128, scaling="yarn", norm=True),
        # four prompts of 2048 tokens taken in one step
        dict(name="append_8192_rows", op="append", cache="fp32", rows=8192, seqs=4, n_heads=32, n_kv=8, hd=128, bs=16,
             far=2048, layout="half", rotary=128, scaling="none", norm=True),
        # ragged prompts of a small model whose rows are no multiple of 32 channels; a third of the head rotated
        dict(name="append_3001_rows_4bit", op="append", cache="mx4", rows=3001, seqs=7, n_heads=6, n_kv=6, hd=48, bs=16,
             far=4096, layout="half", rotary=16, scaling="linear", norm=False),
        # one request of a small model
        dict(name="attend4_1x777_small", op="attend4", seqs=1, rows=1, ctx=777, ragged=False, n_heads=6, n_kv=6, hd=48, bs=16),
        # the decode step this package's benchmark is quoted on
        dict(name="attend4_64x2048", op="attend4", seqs=64, rows=1, ctx=2048, ragged=False, n_heads=32, n_kv=8, hd=128, bs=16),
        # few requests with long contexts
        dict(name="attend4_16x32768", op="attend4", seqs=16, rows=1, ctx=32768, ragged=False, n_heads=32, n_kv=8, hd=128, bs=16),
        # chunks of prompts behind what the cache holds already, none of one length
        dict(name="attend4_chunks_3x1500", op="attend4", seqs=3, rows=1500, ctx=4000, ragged=True, n_heads=32, n_kv=8, hd=128,
             bs=16),
        # the blocks that a decode step has just written to
        dict(name="index_64_newest", op="index", seqs=64, rows=1, ctx=2048, n_kv=8, hd=128, bs=16),
        # the blocks of four prompts of 2048 tokens
        dict(name="index_4x2048_prompt", op="index", seqs=4, rows=2048, ctx=2048, n_kv=8, hd=128, bs=16),
        # one request with an ordinary context, an eighth of it read
        dict(name="sparse_1x8192", op="sparse", seqs=1, ctx=8192, ragged=False, n_heads=32, n_kv=8, hd=128, bs=16, top=64,
             first=1, last=2),
        # few requests with long contexts, a sixteenth read
        dict(name="sparse_16x32768", op="sparse", seqs=16, ctx=32768, ragged=False, n_heads=32, n_kv=8, hd=128, bs=16, top=128,
             first=1, last=4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "append", "attend4", "attend4", "attend4", "index", "sparse", "sparse"))
    n_kv = rng.choice((1, 2, 3, 4, 6, 8, 8, 16))
    n_heads = n_kv * rng.choice((1, 2, 3, 4, 4, 5, 7, 8))
    if op == "append":
        hd = rng.choice((32, 48, 64, 80, 96, 112, 128, 128, 128, 256))
        seqs = _log(rng, 1, 300)
        rows = seqs if rng.random() < 0.5 else _log(rng, 1, 6000) + seqs
        rows = max(seqs, min(rows, 8192 * 48 * 128 // ((n_heads + 2 * n_kv) * hd)))
        scaling = rng.choice(("none", "none", "linear", "ntk", "yarn"))
        cache = rng.choice(("fp32", "mx4"))
        far = min(_log(rng, 64, 100000), (1 << (28 if cache == "fp32" else 31)) // (seqs * n_kv * hd))  # what a pool holds
        return dict(op=op, cache=cache, rows=rows, seqs=seqs, n_heads=n_heads, n_kv=n_kv, hd=hd,
                    bs=rng.choice((16, 16, 32, 64)), far=max(rows // seqs + 1, far),
                    layout=rng.choice(("interleaved", "half")), rotary=rng.choice((hd, hd, hd // 2)), scaling=scaling,
                    norm=rng.random() < 0.5)
    if op == "attend4":
        hd = rng.choice((32, 48, 64, 80, 96, 128, 128, 128, 256))
        if rng.random() < 0.65:  # one row for each sequence
            ctx = _log(rng, 1, 40000)
            most = min(300, 16 * 32768 * 8 * 128 // (ctx * n_kv * hd))
            return dict(op=op, seqs=_log(rng, 1, max(1, most)), rows=1, ctx=ctx, ragged=rng.random() < 0.5, n_heads=n_heads,
                        n_kv=n_kv, hd=hd, bs=rng.choice((16, 16, 32, 64)))
        rows = _log(rng, 2, 1500)
        ctx = rows + _log(rng, 1, 3000)
        while rows * ctx * n_heads * hd > 3 * 1500 * 4000 * 32 * 128:
            rows, ctx = (rows + 1) // 2, (ctx + 1) // 2
        most = min(40, 3 * 1500 * 4000 * 32 * 128 // (rows * ctx * n_heads * hd))
        return dict(op=op, seqs=_log(rng, 1, most), rows=rows, ctx=ctx, ragged=rng.random() < 0.7, n_heads=n_heads, n_kv=n_kv,
                    hd=hd, bs=rng.choice((16, 16, 32, 64)))
    hd = rng.choice((32, 48, 64, 80, 128, 128, 128, 256))
    bs = rng.choice((8, 16, 16, 32, 64))
    if op == "index":
        ctx = _log(rng, 1, 8192)
        most = max(1, min(256, 4 * 2048 * 8 * 128 // (ctx * n_kv * hd)))
        return dict(op=op, seqs=_log(rng, 1, most), rows=rng.choice((1, rng.randint(1, ctx), ctx)), ctx=ctx, n_kv=n_kv, hd=hd,
                    bs=bs)
    ctx = _log(rng, 8, 65536)
    most = max(1, min(256, 16 * 32768 * 8 * 128 // (ctx * n_kv * hd)))
    first, last = rng.randint(0, 2), rng.randint(1, 4)
    return dict(op=op, seqs=_log(rng, 1, most), ctx=ctx, ragged=rng.random() < 0.5, n_heads=n_heads, n_kv=n_kv, hd=hd, bs=bs,
                top=first + last + _log(rng, 1, 128), first=first, last=last)


# ------------------------------------------------------------------------------------------------- lengths of a case
def _lengths(case):
    """Rows and context of every sequence: the case's own, or spread below them where it is ragged."""
    seqs, ctx = case["seqs"], case["ctx"]
    rows = case.get("rows", 1)
    if not case.get("ragged"):
        return [rows] * seqs, [ctx] * seqs
    r = random.Random("%d %d %d" % (seqs, rows, ctx))
    n = [rows if i == 0 else max(1, int(rows * r.uniform(0.2, 1.0))) for i in range(seqs)]
    return n, [max(n[i], ctx if i == 0 else int(ctx * r.uniform(0.1, 1.0))) for i in range(seqs)]


def _append_rows(case):
    """(sequence, position) of every appended row: sequences share the rows, each at the end of a context of its own."""
    rows, seqs = case["rows"], case["seqs"]
    each = [rows // seqs + (i < rows % seqs) for i in range(seqs)]
    r = random.Random("%d %d %d" % (rows, seqs, case["far"]))
    start = [0 if rows > 8 * seqs else r.randint(0, max(0, case["far"] - n)) for n in each]
    seq = [s for s in range(seqs) for _ in range(each[s])]
    pos = [start[s] + i for s in range(seqs) for i in range(each[s])]
    return seq, pos


def _need(lens, bs):
    return [(n + bs - 1) // bs for n in lens]


def _tables(need, gen, extra=3):
    """Block tables dealt from a permutation of a pool with a few blocks to spare; unused entries are 0."""
    total, most = sum(need) + extra, max(need)
    perm = torch.randperm(total, generator=gen, device=DEV, dtype=torch.int32)
    at = torch.arange(most, device=DEV)[None, :]
    n = torch.tensor(need, device=DEV)[:, None]
    first = torch.cumsum(n, 0) - n
    return torch.where(at < n, perm[torch.clamp(first + at, max=total - 1)], 0).to(torch.int32).contiguous(), total


# ------------------------------------------------------------------------------------------------------------- states
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32)


def _keys(gen, rows, n_kv, hd):
    """Key rows as caches hold them: a few channels of each head are several times larger than the rest."""
    return _randn(gen, rows, n_kv, hd) * torch.exp(0.7 * _randn(gen, 1, n_kv, hd))


class _Shared:
    """The stream all operators of this program run on."""

    stream = None


def _stream():
    if _Shared.stream is None:
        _Shared.stream = torch.cuda.Stream()
    return _Shared.stream.cuda_stream


class _Slab:
    """A device buffer of the library as torch sees it; a tensor made from it keeps it, and it keeps the buffer's owner."""

    def __init__(self, owner, ptr, shape):
        self.owner = owner
        self.__cuda_array_interface__ = dict(shape=tuple(shape), typestr="<f4", data=(ptr, False), version=3, strides=None)


def _view(owner, ptr, shape):
    return torch.as_tensor(_Slab(owner, ptr, shape), device=DEV)


def _quantise(x):
    """(codes 0..15, biased exponents) of rows [..., hd] in 64 bits; a group is 32 channels, the last one what is left."""
    hd = x.shape[-1]
    groups = (hd + 31) // 32
    x = torch.nn.functional.pad(x.double(), (0, 32 * groups - hd)).unflatten(-1, (groups, 32))
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m <= 0.875, e - 3, e - 2).clamp(-126, 127)
    e = torch.where(m == 0, torch.full_like(e, -126), e)
    a = torch.ldexp(x.abs(), -e[..., None].double())
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code + 8 * (x < 0)
    return code.flatten(-2)[..., :hd].to(torch.uint8), (e + 127).to(torch.uint8)


def _values(code, exponent):
    """What codes [..., hd] and biased exponents [..., groups] stand for, fp32."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=code.device, dtype=torch.float32)
    scale = torch.ldexp(torch.ones((), device=code.device), exponent.int() - 127)
    return level[code.long()] * scale.repeat_interleave(32, -1)[..., : code.shape[-1]]


def _frequencies(case):
    """Angle per position of every rotated pair and the factor on cos and sin, in 64 bits."""
    r, scaling, factor, trained = case["rotary"], case["scaling"], 8.0, 4096
    i = torch.arange(0, r, 2, device=DEV, dtype=torch.float64)
    if scaling == "ntk" and r > 2:
        return (THETA * factor ** (r / (r - 2))) ** (-i / r), 1.0
    f = THETA ** (-i / r)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        turns = trained * f / (2 * math.pi)  # over the trained context: few are slowed down, many kept
        keep = torch.clamp((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        return (1 - keep) * f / factor + keep * f, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _prepare_append(case, gen):
    rows, H, KV, hd, bs = case["rows"], case["n_heads"], case["n_kv"], case["hd"], case["bs"]
    seq, pos = _append_rows(case)
    need = [0] * case["seqs"]
    for s, p in zip(seq, pos):
        need[s] = max(need[s], p // bs + 1)
    tables, blocks = _tables(need, gen)
    s = dict(case=case, blocks=blocks, tables=tables, q=_randn(gen, rows, H, hd), k=_keys(gen, rows, KV, hd),
             v=_randn(gen, rows, KV, hd), seq=torch.tensor(seq, device=DEV, dtype=torch.int32),
             pos=torch.tensor(pos, device=DEV, dtype=torch.int32))
    s["wq"] = 1 + 0.2 * _randn(gen, hd) if case["norm"] else None
    s["wk"] = 1 + 0.2 * _randn(gen, hd) if case["norm"] else None
    if own:
        import nano_vllm_amd as nv

        s["stream"] = _stream()
        s["rope"] = nv.RotaryTable(hd, case["rotary"], nv.ROPE_HALF if case["layout"] == "half" else nv.ROPE_INTERLEAVED,
                                   THETA, dict(none=nv.ROPE_SCALE_NONE, linear=nv.ROPE_SCALE_LINEAR, ntk=nv.ROPE_SCALE_NTK,
                                               yarn=nv.ROPE_SCALE_YARN)[case["scaling"]], 8.0, 4096)
        s["q_out"] = torch.empty_like(s["q"])
        if case["cache"] == "fp32":
            s["pool"] = nv.PagedKVPool(1, blocks, bs, KV, hd)
            s["slabs"] = tuple(_view(s["pool"], p, (blocks, bs, KV, hd)) for p in s["pool"].layer_ptrs(0))
        else:
            s["pool"] = nv.Mx4KVPool(1, blocks, bs, KV, hd)
            s["k_back"], s["v_back"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    elif case["cache"] == "fp32":
        s["slabs"] = tuple(torch.zeros(blocks, bs, KV, hd, device=DEV) for _ in range(2))
    else:
        s["codes"] = tuple(torch.zeros(blocks, bs, KV, hd, device=DEV, dtype=torch.uint8) for _ in range(2))
        s["exps"] = tuple(torch.zeros(blocks, bs, KV, (hd + 31) // 32, device=DEV, dtype=torch.uint8) for _ in range(2))
    return s


def _prepare_attend4(case, gen):
    H, KV, hd, bs = case["n_heads"], case["n_kv"], case["hd"], case["bs"]
    rows, ctx = _lengths(case)
    tables, blocks = _tables(_need(ctx, bs), gen)
    total, tokens = sum(rows), sum(ctx)
    n = torch.tensor(ctx, device=DEV)
    seq = torch.repeat_interleave(torch.arange(len(ctx), device=DEV), n)
    pos = torch.arange(tokens, device=DEV) - torch.repeat_interleave(torch.cumsum(n, 0) - n, n)
    k, v = _keys(gen, tokens, KV, hd), _randn(gen, tokens, KV, hd)
    off = torch.zeros(len(rows) + 1, device=DEV, dtype=torch.int32)
    off[1:] = torch.cumsum(torch.tensor(rows, device=DEV), 0)
    s = dict(case=case, blocks=blocks, tables=tables, ctx=n.to(torch.int32), off=off, total=total, most_rows=max(rows),
             most_ctx=max(ctx), q=0.6 * _randn(gen, total, H, hd))
    if own:
        import nano_vllm_amd as nv

        s["stream"] = _stream()
        s["pool"] = nv.Mx4KVPool(1, blocks, bs, KV, hd)
        s["out"] = torch.empty_like(s["q"])
        seq32, pos32 = seq.to(torch.int32), pos.to(torch.int32)
        torch.cuda.synchronize()
        nv.norm_rope_append_device(s["pool"], 0, None, tokens, H, None, None, k, v, None, None, EPS, seq32, pos32, tables,
                                   len(ctx), tables.shape[1], s["stream"])
        s["pool"].reserve_workspace(len(ctx), H, max(rows), max(ctx))
        torch.cuda.synchronize()
    else:
        block, at = tables[seq, pos // bs].long(), pos % bs
        s["codes"], s["exps"] = [], []
        for x in (k, v):
            codes = torch.zeros(blocks, bs, KV, hd // 2, device=DEV, dtype=torch.uint8)  # two to a byte
            exps = torch.zeros(blocks, bs, KV, (hd + 31) // 32, device=DEV, dtype=torch.uint8)
            for lo in range(0, tokens, 65536):
                c, e = _quantise(x[lo:lo + 65536])
                codes[block[lo:lo + 65536], at[lo:lo + 65536]] = c[..., 0::2] | (c[..., 1::2] << 4)
                exps[block[lo:lo + 65536], at[lo:lo + 65536]] = e
            s["codes"].append(codes)
            s["exps"].append(exps)
    return s


def _prepare_sparse(case, gen):
    KV, hd, bs = case["n_kv"], case["hd"], case["bs"]
    rows, ctx = _lengths(case)
    tables, blocks = _tables(_need(ctx, bs), gen)
    n = torch.tensor(ctx, device=DEV)
    s = dict(case=case, blocks=blocks, tables=tables, ctx=n.to(torch.int32), most_ctx=max(ctx),
             start=(n - torch.tensor(rows, device=DEV)).to(torch.int32), most_rows=max(rows))
    if case["op"] == "sparse":
        s["q"] = 0.6 * _randn(gen, len(ctx), case["n_heads"], hd)
    shape = (blocks, bs, KV, hd)
    # neighbouring tokens have keys alike: a block's mean, and what each token adds
    mean = _keys(gen, blocks, KV, hd)[:, None]
    if own:
        import nano_vllm_amd as nv

        s["stream"] = _stream()
        s["pool"] = nv.PagedKVPool(1, blocks, bs, KV, hd)
        k, v = (_view(s["pool"], p, shape) for p in s["pool"].layer_ptrs(0))
        torch.add(mean, _randn(gen, *shape), alpha=0.7, out=k)
        v.copy_(_randn(gen, *shape))
        torch.cuda.synchronize()
        s["index"] = nv.BlockIndex(s["pool"])
        zero = torch.zeros_like(s["ctx"])
        if case["op"] == "sparse":
            torch.cuda.synchronize()
            s["index"].update_device(0, len(ctx), tables, tables.shape[1], zero, s["ctx"], max(ctx), s["stream"])
            s["index"].reserve_workspace(len(ctx), case["n_heads"], max(ctx), case["top"])
            s["out"] = torch.empty_like(s["q"])
            s["chosen"] = torch.empty(len(ctx), KV, case["top"], device=DEV, dtype=torch.int32)
        else:
            s["bounds"] = _view(s["index"], s["index"].layer_ptr(0), (blocks, KV, 2, hd))
        torch.cuda.synchronize()
    else:
        s["k"] = torch.add(mean, _randn(gen, *shape), alpha=0.7)
        s["v"] = _randn(gen, *shape)
        s["bounds"] = torch.zeros(blocks, KV, 2, hd, device=DEV)
        if case["op"] == "sparse":
            s["bounds"][:, :, 0], s["bounds"][:, :, 1] = s["k"].amin(1), s["k"].amax(1)
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    return dict(append=_prepare_append, attend4=_prepare_attend4, index=_prepare_sparse, sparse=_prepare_sparse)[case["op"]](case, gen)


# -------------------------------------------------------------------------------------------------------- plain forms
def _rotated(x, weight, case, pos, dtype):
    """Norm and rotation of rows [rows, heads, hd], computed in `dtype` (angles in 64 bits)."""
    x = x.to(dtype)
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.to(dtype)
    freq, factor = _frequencies(case)
    angle = pos.double()[:, None] * freq[None, :]
    c, s = ((factor * t).to(dtype)[:, None, :] for t in (torch.cos(angle), torch.sin(angle)))
    r = case["rotary"]
    turn, rest = x[..., :r], x[..., r:]
    if case["layout"] == "half":
        a, b = turn[..., : r // 2], turn[..., r // 2:]
        return torch.cat((a * c - b * s, a * s + b * c, rest), -1)
    a, b = turn[..., 0::2], turn[..., 1::2]
    return torch.cat((torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2), rest), -1)


def _plain_append(s):
    case, bs = s["case"], s["case"]["bs"]
    pos = s["pos"].long()
    block, at = s["tables"][s["seq"].long(), pos // bs].long(), pos % bs
    q = _rotated(s["q"], s["wq"], case, pos, torch.float32)
    if case["cache"] == "fp32":
        k = _rotated(s["k"], s["wk"], case, pos, torch.float32)
        s["slabs"][0][block, at] = k
        s["slabs"][1][block, at] = s["v"]
        return dict(q=q, k=s["slabs"][0], v=s["slabs"][1])
    k = _rotated(s["k"], s["wk"], case, pos, torch.float64)  # values next to a rounding border
    (kc, ke), (vc, ve) = _quantise(k), _quantise(s["v"])
    s["codes"][0][block, at], s["exps"][0][block, at] = kc, ke
    s["codes"][1][block, at], s["exps"][1][block, at] = vc, ve
    return dict(q=q, k=_values(s["codes"][0][block, at], s["exps"][0][block, at]),
                v=_values(s["codes"][1][block, at], s["exps"][1][block, at]))


def _softmax(x):
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _cached(codes, exps, tables):
    """Rows of a 4-bit cache behind block tables: [seqs, kv heads, tokens, hd] fp32."""
    c = codes[tables.long()].flatten(1, 2)
    c = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    return _values(c, exps[tables.long()].flatten(1, 2)).transpose(1, 2)


def _plain_attend4(s):
    case = s["case"]
    KV, hd, S, R = case["n_kv"], case["hd"], case["seqs"], s["most_rows"]
    k, v = (_cached(s["codes"][i], s["exps"][i], s["tables"]) for i in (0, 1))
    n = (s["off"][1:] - s["off"][:-1]).long()
    at = torch.arange(R, device=DEV)[None, :]
    real = at < n[:, None]
    row = torch.where(real, s["off"][:-1, None].long() + at, 0)
    q = s["q"][row].unflatten(2, (KV, -1)).permute(0, 2, 3, 1, 4)  # [seqs, kv heads, group, rows, hd]
    g = q.shape[2]
    x = torch.matmul(q.reshape(S, KV, g * R, hd), k.transpose(2, 3)).unflatten(2, (g, R)) / math.sqrt(hd)
    limit = s["ctx"][:, None].long() - n[:, None] + at + 1  # a row sees the tokens up to its own
    seen = torch.arange(k.shape[2], device=DEV)[None, None, :] < torch.clamp(limit, min=1)[:, :, None]
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    o = torch.matmul(_softmax(x).reshape(S, KV, g * R, -1), v).unflatten(2, (g, R)).permute(0, 3, 1, 2, 4)
    return o.flatten(2, 3)[real]


def _plain_index(s):
    bs = s["case"]["bs"]
    nb = s["tables"].shape[1]
    b = torch.arange(nb, device=DEV)[None, :]
    hit = (b >= (s["start"] // bs)[:, None]) & (b < ((s["ctx"] + bs - 1) // bs)[:, None])
    at = hit.nonzero()
    block = s["tables"][at[:, 0], at[:, 1]].long()
    held = torch.arange(bs, device=DEV)[None, :] < (s["ctx"].long()[at[:, 0]] - at[:, 1] * bs)[:, None]
    k = s["k"][block]
    s["bounds"][block, :, 0] = torch.where(held[..., None, None], k, math.inf).amin(1)
    s["bounds"][block, :, 1] = torch.where(held[..., None, None], k, -math.inf).amax(1)
    return s["bounds"]


def _choose(score, nblocks, case):
    """The blocks to read, ascending and filled up with -1: first and last ones, then the best; equal scores, lowest first."""
    nb = score.shape[-1]
    b = torch.arange(nb, device=score.device)
    n = nblocks[:, None, None]
    always = (b < case["first"]) | (b >= n - case["last"])
    score = score.masked_fill(always, math.inf).masked_fill(b >= n, -math.inf)
    top = min(case["top"], nb)
    got = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :top]
    got = torch.where(torch.arange(top, device=score.device) < n, got, nb)
    got = torch.sort(got, dim=-1)[0]
    got = torch.nn.functional.pad(got, (0, case["top"] - top), value=nb)
    return torch.where(got < nb, got, -1)


def _plain_sparse(s):
    case, bs = s["case"], s["case"]["bs"]
    KV, hd, S = case["n_kv"], case["hd"], case["seqs"]
    q = s["q"].unflatten(1, (KV, -1))
    bounds = s["bounds"][s["tables"].long()].permute(0, 2, 1, 3, 4).double()  # scores next to each other: 64 bits
    low = torch.matmul(torch.clamp(q, max=0).double(), bounds[..., 0, :].transpose(2, 3))
    high = torch.matmul(torch.clamp(q, min=0).double(), bounds[..., 1, :].transpose(2, 3))
    score = (low + high).amax(2).float()
    nblocks = (s["ctx"].long() + bs - 1) // bs
    chosen = _choose(score, nblocks, case)
    block = s["tables"].long()[torch.arange(S, device=DEV)[:, None, None], chosen.clamp(min=0)]
    head = torch.arange(KV, device=DEV)[None, :, None]
    k = s["k"][block, :, head].flatten(2, 3)
    v = s["v"][block, :, head].flatten(2, 3)
    token = (chosen[..., None] * bs + torch.arange(bs, device=DEV)).flatten(2)
    seen = (token >= 0) & (chosen >= 0).repeat_interleave(bs, -1) & (token < s["ctx"][:, None, None])
    x = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(hd)
    x = x.masked_fill(~seen[:, :, None], -math.inf)
    return dict(out=torch.matmul(_softmax(x), v).flatten(1, 2), chosen=chosen.to(torch.int32))


# ---------------------------------------------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return dict(append=_plain_append, attend4=_plain_attend4, index=_plain_index, sparse=_plain_sparse)[op](s)
    import nano_vllm_amd as nv

    tables, st = s["tables"], s["stream"]
    if op == "append":
        nv.norm_rope_append_device(s["pool"], 0, s["rope"], case["rows"], case["n_heads"], s["q"], s["q_out"], s["k"], s["v"],
                                   s["wq"], s["wk"], EPS, s["seq"], s["pos"], tables, case["seqs"], tables.shape[1], st)
        if case["cache"] == "fp32":
            return dict(q=s["q_out"], k=s["slabs"][0], v=s["slabs"][1])
        s["pool"].read_rows_device(0, case["rows"], s["seq"], s["pos"], tables, case["seqs"], tables.shape[1], s["k_back"],
                                   s["v_back"], st)
        return dict(q=s["q_out"], k=s["k_back"], v=s["v_back"])
    if op == "attend4":
        if s["most_rows"] == 1:
            nv.mx4_decode_device(s["pool"], 0, case["seqs"], case["n_heads"], s["q"], tables, tables.shape[1], s["ctx"],
                                 s["most_ctx"], s["out"], stream=st)
        else:
            nv.mx4_prefill_device(s["pool"], 0, case["seqs"], case["n_heads"], s["total"], s["q"], s["off"], s["most_rows"],
                                  tables, tables.shape[1], s["ctx"], s["most_ctx"], s["out"], stream=st)
        return s["out"]
    if op == "index":
        s["index"].update_device(0, case["seqs"], tables, tables.shape[1], s["start"], s["ctx"], s["most_rows"], st)
        return s["bounds"]
    nv.sparse_decode_device(s["index"], 0, case["seqs"], case["n_heads"], s["q"], tables, tables.shape[1], s["ctx"],
                            s["most_ctx"], case["top"], case["first"], case["last"], s["out"], s["chosen"], stream=st)
    return dict(out=s["out"], chosen=s["chosen"])


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    hd, KV, bs = case["hd"], case["n_kv"], case["bs"]
    H = case.get("n_heads", KV)
    row4 = hd / 2 + (hd + 31) // 32  # bytes of a 4-bit row of one head
    if case["op"] == "append":
        rows = case["rows"]
        kept = 2 * KV * (4 * hd if case["cache"] == "fp32" else row4 + 4 * hd)  # 4 bits: written, and read back as values
        return dict(bytes=rows * (4 * hd * (2 * H + 2 * KV) + kept + 8), flops=rows * (H + KV) * hd * 6)
    rows, ctx = _lengths(case)
    if case["op"] == "attend4":
        pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(rows, ctx))
        return dict(bytes=sum(ctx) * KV * 2 * row4 + 2 * 4 * hd * H * sum(rows) + 4 * sum(_need(ctx, bs)),
                    flops=4 * hd * H * pairs)
    if case["op"] == "index":
        touched = [((c + bs - 1) // bs, (c - n) // bs) for n, c in zip(rows, ctx)]
        blocks = sum(e - b for e, b in touched)
        tokens = sum(c - b * bs for c, (_, b) in zip(ctx, touched))
        return dict(bytes=4 * hd * KV * (tokens + 2 * blocks) + 4 * blocks, flops=2 * hd * KV * tokens)
    need = _need(ctx, bs)
    read = sum(min(c, min(n, case["top"]) * bs) for c, n in zip(ctx, need))
    scored = sum(n for n in need if n > case["top"])
    return dict(bytes=4 * hd * KV * 2 * (read + scored) + 2 * 4 * hd * H * len(ctx) + 4 * sum(need) + 4 * KV * case["top"] * len(ctx),
                flops=4 * hd * H * (read + scored))


# ----------------------------------------------------------------------------------- the operators' definitions, 64 bits
def _exact_turn(x, w, pos, case):
    x = x.double()
    hd, r = case["hd"], case["rotary"]
    if w is not None:
        x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / hd + EPS) * w.double()
    freq, factor = [], 1.0
    for i in range(r // 2):
        f = math.exp(-2.0 * i / r * math.log(THETA))
        if case["scaling"] == "linear":
            f = f / 8.0
        elif case["scaling"] == "ntk" and r > 2:
            f = math.exp(-2.0 * i / r * (math.log(THETA) + r / (r - 2) * math.log(8.0)))
        elif case["scaling"] == "yarn":
            factor = 1.0 + 0.1 * math.log(8.0)
            t = min(1.0, max(0.0, (4096 * f / (2.0 * math.pi) - 1.0) / 31.0))
            f = f * (t + (1.0 - t) / 8.0)
        freq.append(f)
    z = torch.polar(torch.full((len(pos), r // 2), factor, device=DEV, dtype=torch.float64),
                    pos.double()[:, None] * torch.tensor(freq, device=DEV, dtype=torch.float64))[:, None, :]
    y = x.clone()
    first, second = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
    turned = torch.complex(x[..., first], x[..., second]) * z
    y[..., first], y[..., second] = turned.real, turned.imag
    return y


def _exact_round4(x):
    """Nearest value of the 4-bit format for rows [..., hd], by search over its sixteen levels."""
    got = torch.empty_like(x)
    level = torch.tensor(LEVELS, device=DEV, dtype=torch.float64)
    even = torch.tensor((0, 2, 4, 6, 1, 3, 5, 7), device=DEV)  # argmin takes the first: even codes go first on a tie
    for lo in range(0, x.shape[-1], 32):
        part = x[..., lo:lo + 32]
        most = part.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(torch.clamp(most, min=1e-300) / 7.0))
        e = torch.where(7.0 * torch.exp2(e - 1) >= most, e - 1, e)
        e = torch.where(7.0 * torch.exp2(e) < most, e + 1, e).clamp(-126, 127)
        near = (part.abs() / torch.exp2(e)).clamp(max=6.0)
        which = even[(near[..., None] - level[even]).abs().argmin(-1)]
        got[..., lo:lo + 32] = torch.sign(part) * level[which] * torch.exp2(e)
    return got


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    hd, KV, bs = case["hd"], case["n_kv"], case["bs"]
    if case["op"] == "append":
        q, k = _exact_turn(s["q"], s["wq"], s["pos"], case), _exact_turn(s["k"], s["wk"], s["pos"], case)
        if case["cache"] == "mx4":
            return dict(q=q, k=_exact_round4(k), v=_exact_round4(s["v"].double()))
        slabs = [torch.zeros(t.shape, device=DEV, dtype=torch.float64) for t in s["slabs"]]
        slot = s["tables"].long()[s["seq"].long(), s["pos"].long() // bs] * bs + s["pos"].long() % bs
        for slab, rows in zip(slabs, (k, s["v"].double())):
            slab.view(-1, KV, hd)[slot] = rows
        return dict(q=q, k=slabs[0], v=slabs[1])
    if case["op"] == "index":
        got = torch.zeros(s["bounds"].shape, device=DEV, dtype=torch.float64)
        for i in range(case["seqs"]):
            b, e = int(s["start"][i]), int(s["ctx"][i])
            for j in range(b // bs, (e + bs - 1) // bs):
                p = int(s["tables"][i, j])
                rows = s["k"][p, : min(bs, e - j * bs)].double()
                got[p, :, 0], got[p, :, 1] = rows.min(0)[0], rows.max(0)[0]
        return got
    H = case["n_heads"]
    g = H // KV
    out = torch.empty(s["q"].shape, device=DEV, dtype=torch.float64)
    if case["op"] == "attend4":
        off = s["off"].tolist()
        for i in range(case["seqs"]):
            T, n = int(s["ctx"][i]), off[i + 1] - off[i]
            ids = s["tables"][i, : (T + bs - 1) // bs].long()
            x = []
            for codes, exps in zip(s["codes"], s["exps"]):
                c = codes[ids].flatten(0, 1)[:T].int()
                c = torch.stack((c % 16, torch.div(c, 16, rounding_mode="floor")), -1).flatten(-2)
                mag = torch.tensor(LEVELS, device=DEV, dtype=torch.float64)[(c % 8).long()]
                e = exps[ids].flatten(0, 1)[:T].double() - 127
                e = e[..., torch.arange(hd, device=DEV) // 32]
                x.append(mag * torch.where(c >= 8, -1.0, 1.0) * torch.exp2(e))
            seen = torch.arange(T, device=DEV)[None, :] <= torch.arange(T - n, T, device=DEV)[:, None]
            for h in range(H):
                a = s["q"][off[i]:off[i + 1], h].double() @ x[0][:, h // g].T / math.sqrt(hd)
                out[off[i]:off[i + 1], h] = torch.softmax(torch.where(seen, a, -math.inf), -1) @ x[1][:, h // g]
        return out
    for i in range(case["seqs"]):
        T = int(s["ctx"][i])
        nb = (T + bs - 1) // bs
        ids = s["tables"][i, :nb].long()
        lim = s["bounds"][ids].double()
        for j in range(KV):
            q = s["q"][i, j * g:(j + 1) * g].double()
            score = (q[:, None, :] * torch.where(q[:, None, :] > 0, lim[None, :, j, 1], lim[None, :, j, 0])).sum(-1).max(0)[0].float()
            must = sorted(set(range(min(case["first"], nb))) | set(range(max(0, nb - case["last"]), nb)))
            rest = torch.ones(nb, device=DEV, dtype=torch.bool)
            rest[must] = False
            others = rest.nonzero().flatten()
            order = torch.sort(-score[others].double(), stable=True)[1][: max(0, min(nb, case["top"]) - len(must))]
            keep = torch.cat((torch.tensor(must, device=DEV), others[order])).sort()[0]
            token = (keep[:, None] * bs + torch.arange(bs, device=DEV)).flatten()
            token = token[token < T]
            k, v = (s[t][ids[token // bs], token % bs, j].double() for t in ("k", "v"))
            out[i, j * g:(j + 1) * g] = torch.softmax(q @ k.T / math.sqrt(hd), -1) @ v
    return dict(out=out, chosen=None)
