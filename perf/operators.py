"""The operators beside the attention forward, as cases that can be timed and compared: its gradient (training), and a
paged key-value cache with the attention of new tokens that reads it (generation).

  backward  dQ, dK, dV of the attention forward from Q, K, V, its output O, its log-sum-exp and dO. The probabilities are
            taken again from the scores and the log-sum-exp: P = exp(s - lse), dS = P * (dO V^T - rowsum(dO * O)),
            dQ = scale * dS K, dK = scale * dS^T Q, dV = P^T dO.
  append    new keys and values of every sequence go to their places in the pages of the cache, keys (and the queries
            beside them) rotated by the angles of their positions on the way.
  decode    softmax(scale * q K^T + mask) V of the newest token, or the newest few, of every sequence over the keys and
            values that the sequence has in the cache, and its log-sum-exp.

Each has a plain form of elementary torch operations in 32 bits, rounded once at the end, and an evaluation of its
definition in 64 bits (`exact`) that shares no code with the plain form. With `own` set, `run` makes the calls of the
package instead.
"""
import importlib
import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _package():
    return importlib.import_module("flash-attn-rtx5060_b200")


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _backward(name, batch, heads, seqlen, head_dim, causal, window_left=-1, window_right=-1, alibi=False, spread=1.0,
              grad=1.0):
    """spread: standard deviation of the scaled scores; grad: of the elements of dO."""
    return {"name": name, "op": "backward", "batch": batch, "heads": heads, "seqlen": seqlen, "head_dim": head_dim,
            "causal": causal, "window_left": window_left, "window_right": window_right, "alibi": alibi, "spread": spread,
            "grad": grad}


def _append(name, batch, tokens, q_heads, kv_heads, head_dim, page_size, past, dtype, rotary_dim, interleaved=False,
            padded=False, token_major=False):
    """past: the longest that a sequence is before the call; padded: sequences bring up to `tokens` tokens, not all of
    them; token_major: pages hold [token][head], not [head][token]."""
    return {"name": name, "op": "append", "batch": batch, "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page_size": page_size, "past": past, "dtype": dtype, "rotary_dim": rotary_dim,
            "interleaved": interleaved, "padded": padded, "token_major": token_major}


def _decode(name, batch, tokens, q_heads, kv_heads, head_dim, page_size, longest, dtype, ragged=True, window_left=-1,
            alibi=False, spread=1.0, token_major=False):
    """longest: of the sequences' lengths; ragged: lengths from an eighth of it, else all are that long."""
    return {"name": name, "op": "decode", "batch": batch, "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page_size": page_size, "longest": longest, "dtype": dtype, "ragged": ragged,
            "window_left": window_left, "alibi": alibi, "spread": spread, "token_major": token_major}


def listed():
    return [
        # One small layer of the benchmark's smallest configuration: launches and latency.
        _backward("backward_small_d64", 1, 4, 512, 64, False),
        # A batch of ragged encoder inputs; loss gradients as they come without loss scaling.
        _backward("backward_ragged_d64", 8, 12, 1000, 64, False, spread=2.0, grad=2.0 ** -9),
        # Long decoder context with 128-wide heads, the library's main configuration.
        _backward("backward_decoder_d128", 2, 32, 8192, 128, True),
        # Sliding-window decoder.
        _backward("backward_window_d128", 4, 16, 16384, 128, True, window_left=1024, grad=2.0 ** -5),
        # ALiBi-biased decoder.
        _backward("backward_alibi_d64", 2, 16, 4096, 64, True, alibi=True),
        # One step of generation, a few sequences: what counts is the latency of the launch.
        _append("append_step_d128", 4, 1, 32, 8, 128, 16, 2000, "fp16", 128),
        # Prompts of a padded batch enter the cache; a quarter of the head is rotated, in pairs of neighbours.
        _append("append_prompts_bf16_d128", 8, 2048, 32, 8, 128, 64, 0, "bf16", 32, interleaved=True, padded=True,
                token_major=True),
        # One short sequence without shared heads, on the smallest head.
        _decode("decode_one_d64", 1, 1, 4, 4, 64, 16, 512, "fp16", ragged=False),
        # A batch that is being served: sequences of many lengths, small pages, four queries to a key head.
        _decode("decode_batch_d128", 32, 1, 32, 8, 128, 16, 8192, "fp16", spread=2.0),
        # A single long document: few rows, all the work along the cache.
        _decode("decode_long_bf16_d128", 1, 1, 32, 8, 128, 64, 131072, "bf16", ragged=False, spread=2.0),
        # The largest pool: many long sequences.
        _decode("decode_many_d128", 64, 1, 32, 8, 128, 64, 32768, "fp16", token_major=True),
        # Four guessed tokens a sequence are checked in one call, sliding window and ALiBi, every query its own key head.
        _decode("decode_guesses_d64", 16, 4, 16, 16, 64, 32, 4096, "bf16", window_left=2047, alibi=True),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["backward", "append", "decode", "backward", "decode"])
    limits = {"backward": (3e12, 2.1e9), "append": (1e15, 3.2e8), "decode": (1e15, 4.8e9)}[op]
    while True:
        head_dim = rng.choice([64, 128])
        if op == "backward":
            seqlen = log_int(16, 16384)
            if seqlen >= 256 and rng.random() < 0.4:
                seqlen -= seqlen % 128
            causal, wl, wr = rng.random() < 0.6, -1, -1
            if rng.random() < 0.3:
                wl = log_int(8, max(8, seqlen // 2))
                if not causal and rng.random() < 0.7:
                    wr = log_int(8, max(8, seqlen // 2))
            case = _backward("", log_int(1, 8), log_int(1, 32), seqlen, head_dim, causal, wl, wr,
                             alibi=rng.random() < 0.2, spread=rng.choice([1.0, 1.0, 2.0]),
                             grad=2.0 ** -rng.randint(0, 10))
        else:
            kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
            q_heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 7, 8])
            page = rng.choice([8, 16, 16, 24, 32, 64, 128, 256])
            dtype = rng.choice(["fp16", "bf16"])
            if op == "append":
                tokens = 1 if rng.random() < 0.5 else log_int(2, 2048)
                case = _append("", log_int(1, 128), tokens, q_heads, kv_heads, head_dim, page, log_int(1, 8192), dtype,
                               rng.choice([0, 32, head_dim // 2, head_dim, head_dim]), rng.random() < 0.4,
                               rng.random() < 0.4, rng.random() < 0.5)
            else:
                tokens = 1 if rng.random() < 0.7 else rng.randint(2, 8)
                case = _decode("", log_int(1, 128), tokens, q_heads, kv_heads, head_dim, page, log_int(16, 131072), dtype,
                               rng.random() < 0.8, log_int(16, 4096) if rng.random() < 0.2 else -1, rng.random() < 0.2,
                               rng.choice([1.0, 2.0]), rng.random() < 0.5)
        w = work(case)
        pool = 4 * _pool_pages(case) * case["page_size"] * case["kv_heads"] * head_dim if op != "backward" else 0
        if w["flops"] <= limits[0] and w["bytes"] <= limits[1] and pool <= (9e9 if op == "decode" else 2.5e9):
            del case["name"]
            return case


# ---------------------------------------------------------------------------------------------------------------------
# the batch of a case: lengths before and after the call, new tokens
# ---------------------------------------------------------------------------------------------------------------------
def _spread_over(n, lo, hi):
    """n lengths from lo to hi, in an order that is neither rising nor falling; the last of a larger batch is lo."""
    if n == 1:
        return [hi]
    step = next(s for s in (7, 5, 3, 2, 1) if math.gcd(s, n) == 1)
    return [lo + (hi - lo) * ((step * i) % n) // (n - 1) for i in range(1, n + 1)]


def _batch(case):
    """(length of every sequence with its new tokens, number of new tokens of every sequence)."""
    n, t = case["batch"], case["tokens"]
    if case["op"] == "append":
        counts = _spread_over(n, min(1, t), t) if case["padded"] else [t] * n
        return [p + c for p, c in zip(_spread_over(n, case["past"] // 4, case["past"]), counts)], counts
    longest = max(case["longest"], t)
    lengths = _spread_over(n, max(t, longest // 8), longest) if case["ragged"] else [longest] * n
    return lengths, [t] * n


def _pages_of(case):
    return [-(-length // case["page_size"]) for length in _batch(case)[0]]


def _pool_pages(case):
    need = sum(_pages_of(case))
    return need + need // 16 + 1


def _first_key(case, position):
    return 0 if case["window_left"] < 0 else max(0, position - case["window_left"])


def _visible(case):
    """Of one head: the (query, key) pairs and the keys that any query sees."""
    n, wl, wr = case["seqlen"], case["window_left"], 0 if case["causal"] else case["window_right"]
    left, right = (n - 1 if w < 0 else min(w, n - 1) for w in (wl, wr))
    return n + left * n - left * (left + 1) // 2 + right * n - right * (right + 1) // 2


def work(case):
    d = case["head_dim"]
    if case["op"] == "backward":
        bh, n = case["batch"] * case["heads"], case["seqlen"]
        # five products over the visible pairs: scores, dO V^T, dV, dK, dQ
        return {"bytes": 8 * 2 * bh * n * d + 4 * bh * n, "flops": 10 * d * bh * _visible(case)}
    lengths, counts = _batch(case)
    new, hq, hkv = sum(counts), case["q_heads"], case["kv_heads"]
    if case["op"] == "append":
        rows = 2 * 2 * d * new * (2 * hkv + (hq if case["rotary_dim"] else 0))  # read and written, 2 bytes an element
        angles = 4 * case["rotary_dim"] * min(new, max(lengths))
        return {"bytes": rows + angles + 8 * case["batch"], "flops": 3 * case["rotary_dim"] * new * (hq + hkv)}
    keys = sum(length - _first_key(case, length - t) for length, t in zip(lengths, counts))
    pairs = sum(p + 1 - _first_key(case, p) for length, t in zip(lengths, counts) for p in range(length - t, length))
    nbytes = 2 * 2 * d * hkv * keys + 2 * 2 * d * hq * new + 4 * hq * new + 4 * sum(_pages_of(case)) + 4 * case["batch"]
    return {"bytes": nbytes, "flops": 4 * d * hq * pairs}


# ---------------------------------------------------------------------------------------------------------------------
# what a caller holds before the call
# ---------------------------------------------------------------------------------------------------------------------
def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda", dtype=torch.float32)


def _angles(positions, rotary_dim):
    """cos and sin of position * 10000^(-2i / rotary_dim), one row a position: all cosines, then all sines."""
    i = torch.arange(rotary_dim // 2, device="cuda", dtype=torch.float64)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-2.0 * i / rotary_dim)
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    d = case["head_dim"]

    def normal(*shape, dtype=torch.float16, std=1.0):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
        return x.mul_(std) if std != 1.0 else x

    state = {"case": case}
    if case["op"] == "backward":
        shape = (case["batch"], case["heads"], case["seqlen"], d)
        state.update(q=normal(*shape, std=case["spread"]), k=normal(*shape), v=normal(*shape),
                     dout=normal(*shape, std=case["grad"]), slopes=_slopes(case["heads"]) if case["alibi"] else None)
        state["out"], state["lse"] = _plain_forward(state)
        return state

    dtype, hq, hkv, t, ps = _TYPES[case["dtype"]], case["q_heads"], case["kv_heads"], case["tokens"], case["page_size"]
    lengths, counts = _batch(case)
    pool, pages = _pool_pages(case), _pages_of(case)
    shape = (pool, ps, hkv, d) if case["token_major"] else (pool, hkv, ps, d)
    std = 1.0 if case["op"] == "decode" else 0.5
    for name in ("k_pages", "v_pages"):
        x = normal(*shape, dtype=dtype, std=std)
        state[name] = x.transpose(1, 2) if case["token_major"] else x
    order = torch.randperm(pool, generator=gen, device="cuda").tolist()
    table = torch.full((case["batch"], max(max(pages), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    state.update(page_table=table.cuda(), lengths=torch.tensor(lengths, dtype=torch.int32).cuda(), host_lengths=lengths,
                 counts=None, host_counts=counts)
    # queries, keys and values of the new tokens as one projection leaves them: [batch][token][head], read as views
    qkv = normal(case["batch"], t, hq + 2 * hkv, d, dtype=dtype).transpose(1, 2)
    state["q"] = qkv[:, :hq]
    if case["op"] == "append":
        state.update(k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:])
        if case["padded"]:
            state["counts"] = torch.tensor(counts, dtype=torch.int32).cuda()
        state["rotary"] = _angles(max(lengths), case["rotary_dim"]) if case["rotary_dim"] else None
    else:
        if case["spread"] != 1.0:
            state["q"] = state["q"] * case["spread"]
        state["slopes"] = _slopes(hq) if case["alibi"] else None
    return state


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _blocks(case):
    """Blocks of heads and query rows whose scores fit 2^28 elements, with the keys that the rows see."""
    n, bh = case["seqlen"], case["batch"] * case["heads"]
    wl, wr = case["window_left"], 0 if case["causal"] else case["window_right"]
    rows = n if wl < 0 and n <= 16384 else min(n, 2048)
    heads = max(1, min(bh, (1 << 28) // (rows * n)))
    for h in range(0, bh, heads):
        for r0 in range(0, n, rows):
            r1 = min(n, r0 + rows)
            lo = 0 if wl < 0 else max(0, r0 - wl)
            hi = n if wr < 0 else min(n, r1 + wr)
            yield slice(h, min(bh, h + heads)), slice(r0, r1), slice(lo, hi)


def _plain_scores(state, q, k, heads, rows, keys):
    case = state["case"]
    s = torch.matmul(q, k.transpose(1, 2)) * (1.0 / math.sqrt(case["head_dim"]))
    gap = (torch.arange(keys.start, keys.stop, device="cuda")[None, :] -
           torch.arange(rows.start, rows.stop, device="cuda")[:, None])
    if case["alibi"]:
        per_head = state["slopes"].repeat(case["batch"])[heads]
        s = s - per_head[:, None, None] * gap.abs().float()
    wr = 0 if case["causal"] else case["window_right"]
    if case["window_left"] >= 0:
        s = s.masked_fill(gap < -case["window_left"], -math.inf)
    if wr >= 0:
        s = s.masked_fill(gap > wr, -math.inf)
    return s


def _plain_forward(state):
    case = state["case"]
    shape = state["q"].shape
    q, k, v = (state[x].view(-1, shape[2], shape[3]) for x in "qkv")
    out = torch.empty(q.shape, device="cuda", dtype=torch.float16)
    lse = torch.empty(q.shape[:2], device="cuda", dtype=torch.float32)
    for heads, rows, keys in _blocks(case):
        s = _plain_scores(state, q[heads, rows].float(), k[heads, keys].float(), heads, rows, keys)
        top = s.amax(dim=2, keepdim=True)
        p = (s - top).exp()
        total = p.sum(dim=2, keepdim=True)
        out[heads, rows] = (torch.matmul(p, v[heads, keys].float()) / total).half()
        lse[heads, rows] = (top + total.log()).squeeze(2)
    return out.view(shape), lse.view(shape[:3])


def _plain_backward(state):
    case = state["case"]
    shape = state["q"].shape
    q, k, v, out, dout = (state[x].view(-1, shape[2], shape[3]) for x in ("q", "k", "v", "out", "dout"))
    lse = state["lse"].view(-1, shape[2])
    dq, dk, dv = (torch.zeros(q.shape, device="cuda", dtype=torch.float32) for _ in range(3))
    for heads, rows, keys in _blocks(case):
        qb, kb, vb = q[heads, rows].float(), k[heads, keys].float(), v[heads, keys].float()
        gb = dout[heads, rows].float()
        p = (_plain_scores(state, qb, kb, heads, rows, keys) - lse[heads, rows, None]).exp()
        delta = (gb * out[heads, rows].float()).sum(dim=2, keepdim=True)
        dv[heads, keys] += torch.matmul(p.transpose(1, 2), gb)
        ds = p * (torch.matmul(gb, vb.transpose(1, 2)) - delta) * (1.0 / math.sqrt(case["head_dim"]))
        dq[heads, rows] += torch.matmul(ds, kb)
        dk[heads, keys] += torch.matmul(ds.transpose(1, 2), qb)
    return tuple(x.half().view(shape) for x in (dq, dk, dv))


def _plain_rotate(x, table, interleaved):
    """x: [head][token][d] in 32 bits; table: one row of cosines and sines a token."""
    half = table.shape[1] // 2
    cos, sin = table[:, :half], table[:, half:]
    part = x[..., :2 * half]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = part[..., :half], part[..., half:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def _plain_append(state):
    case = state["case"]
    turned = torch.zeros(state["q"].shape, device="cuda", dtype=state["q"].dtype) if case["rotary_dim"] else None
    for b, (length, count) in enumerate(zip(state["host_lengths"], state["host_counts"])):
        at = torch.arange(length - count, length, device="cuda")
        page, slot = state["page_table"][b, at // case["page_size"]].long(), at % case["page_size"]
        k = state["k"][b, :, :count]
        if case["rotary_dim"]:
            angles = state["rotary"][at]
            k = _plain_rotate(k.float(), angles, case["interleaved"]).to(k.dtype)
            turned[b, :, :count] = _plain_rotate(state["q"][b, :, :count].float(), angles, case["interleaved"]).to(k.dtype)
        state["k_pages"][page, :, slot] = k.transpose(0, 1)
        state["v_pages"][page, :, slot] = state["v"][b, :, :count].transpose(0, 1)
    new = [state["k_pages"], state["v_pages"]]
    return new + [turned] if turned is not None else new


def _plain_decode(state):
    case = state["case"]
    hq, hkv, t, d = case["q_heads"], case["kv_heads"], case["tokens"], case["head_dim"]
    out = torch.zeros((case["batch"], hq, t, d), device="cuda", dtype=state["q"].dtype)
    lse = torch.full((case["batch"], hq, t), -math.inf, device="cuda", dtype=torch.float32)
    for b, length in enumerate(state["host_lengths"]):
        lo = _first_key(case, length - t)
        ps = case["page_size"]
        pages = state["page_table"][b, lo // ps:-(-length // ps)].long()
        skip = lo - lo // ps * ps

        def dense(pool):  # [kv_head][key][d]
            return pool[pages].transpose(0, 1).reshape(hkv, -1, d)[:, skip:skip + length - lo].float()

        q = state["q"][b].float().reshape(hkv, hq // hkv * t, d)
        s = torch.matmul(q, dense(state["k_pages"]).transpose(1, 2)) * (1.0 / math.sqrt(d))
        s = s.view(hq, t, length - lo)
        gap = (torch.arange(lo, length, device="cuda")[None, :] -
               torch.arange(length - t, length, device="cuda")[:, None])
        if case["alibi"]:
            s = s - state["slopes"][:, None, None] * gap.abs().float()
        s = s.masked_fill(gap > 0, -math.inf)
        if case["window_left"] >= 0:
            s = s.masked_fill(gap < -case["window_left"], -math.inf)
        top = s.amax(dim=2, keepdim=True)
        p = (s - top).exp()
        total = p.sum(dim=2, keepdim=True)
        o = torch.matmul(p.view(hkv, hq // hkv * t, -1), dense(state["v_pages"])).view(hq, t, d) / total
        out[b] = o.to(out.dtype)
        lse[b] = (top + total.log()).squeeze(2)
    return out, lse


def run(state):
    case = state["case"]
    if not own:
        return {"backward": _plain_backward, "append": _plain_append, "decode": _plain_decode}[case["op"]](state)
    fa = _package()
    if case["op"] == "backward":
        return fa.attention_backward(state["q"], state["k"], state["v"], state["out"], state["lse"], state["dout"],
                                     causal=case["causal"], window_left=case["window_left"],
                                     window_right=case["window_right"], alibi_slopes=state["slopes"])
    if case["op"] == "append":
        if not case["rotary_dim"]:
            fa.cache_append(state["k"], state["v"], state["k_pages"], state["v_pages"], state["page_table"],
                            state["lengths"], counts=state["counts"])
            return [state["k_pages"], state["v_pages"]]
        turned = fa.cache_append(state["k"], state["v"], state["k_pages"], state["v_pages"], state["page_table"],
                                 state["lengths"], counts=state["counts"], q=state["q"], rotary=state["rotary"],
                                 interleaved=case["interleaved"])
        return [state["k_pages"], state["v_pages"], turned]
    return fa.attention_decode(state["q"], state["k_pages"], state["v_pages"], state["page_table"], state["lengths"],
                               window_left=case["window_left"], alibi_slopes=state["slopes"], return_lse=True)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_backward(case, state):
    """Block of keys by block of keys: P and dS of the rows that see any of them, from the definitions."""
    n, d, wl, wr = case["seqlen"], case["head_dim"], case["window_left"], 0 if case["causal"] else case["window_right"]
    grads = [torch.zeros(state["q"].shape, dtype=torch.float64) for _ in range(3)]
    step = max(64, min(n, (1 << 26) // n))
    for b in range(case["batch"]):
        for h in range(case["heads"]):
            q, k, v, o, g = (state[x][b, h].to(torch.float64) for x in ("q", "k", "v", "out", "dout"))
            lse, delta = state["lse"][b, h].to(torch.float64), torch.einsum("id,id->i", g, o)
            dq = torch.zeros_like(q)
            for j0 in range(0, n, step):
                j1 = min(n, j0 + step)
                i0 = 0 if wr < 0 else max(0, j0 - wr)
                i1 = n if wl < 0 else min(n, j1 + wl)
                i, j = torch.arange(i0, i1, device="cuda")[:, None], torch.arange(j0, j1, device="cuda")[None, :]
                logits = torch.einsum("id,jd->ij", q[i0:i1], k[j0:j1]) / d ** 0.5
                if case["alibi"]:
                    logits -= (i - j).abs() * state["slopes"][h].item()
                hidden = torch.zeros_like(logits, dtype=torch.bool)
                if wl >= 0:
                    hidden |= j < i - wl
                if wr >= 0:
                    hidden |= j > i + wr
                p = torch.exp(logits - lse[i0:i1, None])
                p[hidden] = 0.0
                ds = p * (torch.einsum("id,jd->ij", g[i0:i1], v[j0:j1]) - delta[i0:i1, None]) / d ** 0.5
                dq[i0:i1] += torch.einsum("ij,jd->id", ds, k[j0:j1])
                grads[1][b, h, j0:j1] = torch.einsum("ij,id->jd", ds, q[i0:i1]).cpu()
                grads[2][b, h, j0:j1] = torch.einsum("ij,id->jd", p, g[i0:i1]).cpu()
            grads[0][b, h] = dq.cpu()
    return tuple(grads)


def _exact_append(case, state):
    """Every pair of elements is a complex number, turned by cos + i sin of its position."""
    k_pages, v_pages = (state[x].to(torch.float64) for x in ("k_pages", "v_pages"))
    r, half = case["rotary_dim"], case["rotary_dim"] // 2
    if r:
        turn = torch.complex(state["rotary"][:, :half].double(), state["rotary"][:, half:].double())
        first = torch.arange(0, r, 2, device="cuda") if case["interleaved"] else torch.arange(half, device="cuda")
        second = first + (1 if case["interleaved"] else half)

    def turned(x, position):  # x: [head][d]
        x = x.to(torch.float64)
        if r:
            z = torch.complex(x[:, first], x[:, second]) * turn[position]
            x[:, first], x[:, second] = z.real, z.imag
        return x

    table = state["page_table"].tolist()
    q_new = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    lengths, counts = _batch(case)
    if sum(counts) > 40000:
        return None
    for b, (length, count) in enumerate(zip(lengths, counts)):
        for i in range(count):
            position = length - count + i
            page, slot = table[b][position // case["page_size"]], position % case["page_size"]
            k_pages[page, :, slot] = turned(state["k"][b, :, i], position)
            v_pages[page, :, slot] = state["v"][b, :, i].to(torch.float64)
            if r:
                q_new[b, :, i] = turned(state["q"][b, :, i], position)
    return [k_pages, v_pages, q_new] if r else [k_pages, v_pages]


def _exact_decode(case, state):
    hq, group, t, d = case["q_heads"], case["q_heads"] // case["kv_heads"], case["tokens"], case["head_dim"]
    out = torch.zeros((case["batch"], hq, t, d), dtype=torch.float64)
    lse = torch.full((case["batch"], hq, t), -math.inf, dtype=torch.float64)
    lengths = _batch(case)[0]
    slots = torch.arange(max(lengths), device="cuda")
    for b, length in enumerate(lengths):
        page, slot = state["page_table"][b, slots[:length] // case["page_size"]].long(), slots[:length] % case["page_size"]
        for kv in range(case["kv_heads"]):
            k, v = (state[x][page, kv, slot].to(torch.float64) for x in ("k_pages", "v_pages"))
            for i in range(t):
                last = length - t + i
                begin = _first_key(case, last)
                heads = slice(kv * group, (kv + 1) * group)
                logits = torch.einsum("hd,jd->hj", state["q"][b, heads, i].to(torch.float64), k[begin:last + 1]) / d ** 0.5
                if case["alibi"]:
                    logits -= state["slopes"][heads, None].double() * (last - slots[begin:last + 1])
                out[b, heads, i] = torch.einsum("hj,jd->hd", torch.softmax(logits, dim=1), v[begin:last + 1]).cpu()
                lse[b, heads, i] = torch.logsumexp(logits, dim=1).cpu()
    return out, lse


def exact(case, seed):
    state = prepare(case, seed)
    return {"backward": _exact_backward, "append": _exact_append, "decode": _exact_decode}[case["op"]](case, state)
