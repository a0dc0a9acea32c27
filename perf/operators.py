"""Cases of the speculative-decoding operators: attention of new tokens over a paged cache and the store that fills it,
the DeltaNet step over a span of tokens, and the verification of drafted tokens.

Every operator takes packed token rows: sequence b owns rows start[b] .. start[b + 1] - 1.  `run` computes them in plain
torch, or, where `own` is true, through the framework's entry points.  Sizes follow the Qwen3.5-0.8B layout that the
framework serves (8 query heads, 2 key/value heads, head size 256, rotary 64; 16 DeltaNet heads of 128; vocabulary
248320) beside generic ones."""
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


# ---- cases --------------------------------------------------------------------------------------------------------

def listed():
    qwen = {"q_heads": 8, "kv_heads": 2, "head_dim": 256}
    return [
        # a chat turn's next token: one sequence, where latency is all
        {"name": "attend_one_token", "op": "attend", "batch": 1, "q_lo": 1, "q_hi": 1, "kv_lo": 577, "kv_hi": 577,
         "page": 16, "dtype": "f16", "gated": True, **qwen},
        # a full server's decode step: 256 sequences at different lengths
        {"name": "attend_decode_256", "op": "attend", "batch": 256, "q_lo": 1, "q_hi": 1, "kv_lo": 65, "kv_hi": 1150,
         "page": 64, "dtype": "f16", "gated": True, **qwen},
        # four drafted tokens and the last accepted one, verified at once for 64 sequences
        {"name": "attend_drafts_64", "op": "attend", "batch": 64, "q_lo": 5, "q_hi": 5, "kv_lo": 130, "kv_hi": 4000,
         "page": 16, "dtype": "bf16", "gated": True, **qwen},
        # a chunk of a long prompt over what the cache holds of it already
        {"name": "attend_chunk_long", "op": "attend", "batch": 1, "q_lo": 2048, "q_hi": 2048, "kv_lo": 16384,
         "kv_hi": 16384, "page": 64, "dtype": "f16", "gated": True, **qwen},
        # several fresh prompts of odd lengths, ungated heads of 128
        {"name": "attend_prompts_128", "op": "attend", "batch": 8, "q_lo": 301, "q_hi": 1021, "kv_lo": 301,
         "kv_hi": 1021, "page": 32, "dtype": "bf16", "gated": False, "q_heads": 16, "kv_heads": 4, "head_dim": 128},
        # the store beside attend_drafts_64: 320 rows
        {"name": "prep_drafts_64", "op": "prep", "batch": 64, "q_lo": 5, "q_hi": 5, "kv_lo": 130, "kv_hi": 600,
         "page": 16, "dtype": "bf16", "rotary": 64, "gated": True, **qwen},
        # the store of four prompts of about a thousand tokens
        {"name": "prep_prompts", "op": "prep", "batch": 4, "q_lo": 901, "q_hi": 1150, "kv_lo": 1200, "kv_hi": 1700,
         "page": 64, "dtype": "f16", "rotary": 64, "gated": True, **qwen},
        # the DeltaNet layers of a verification: outputs of five tokens, the state left alone
        {"name": "span_verify_64", "op": "span", "batch": 64, "n_lo": 5, "n_hi": 5, "heads": 16, "commit": False},
        # after it: the state moved on by the accepted tokens of each sequence
        {"name": "span_commit_64", "op": "span", "batch": 64, "n_lo": 5, "n_hi": 5, "heads": 16, "commit": True},
        # one sequence's drafts, greedy
        {"name": "verify_greedy_one", "op": "verify", "batch": 1, "rows_lo": 5, "rows_hi": 5, "vocab": 248320,
         "dtype": "f16", "probs": False, "greedy": True},
        # sampled drafts of 64 sequences against a draft model's probabilities
        {"name": "verify_sampled_64", "op": "verify", "batch": 64, "rows_lo": 5, "rows_hi": 5, "vocab": 248320,
         "dtype": "f16", "probs": True, "greedy": False},
        # drafts without probabilities (looked up in the prompt) of uneven number, a small vocabulary
        {"name": "verify_lookup_200", "op": "verify", "batch": 200, "rows_lo": 1, "rows_hi": 9, "vocab": 32003,
         "dtype": "bf16", "probs": False, "greedy": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "prep", "span", "verify"])
    while True:
        if op in ("attend", "prep"):
            head_dim = rng.choice([64, 128, 256, 256])
            kv_heads = rng.choice([1, 2, 2, 4])
            c = {"op": op, "batch": _log_int(rng, 1, 256), "q_lo": 1, "q_hi": 1, "kv_lo": 1, "kv_hi": 1,
                 "page": rng.choice([8, 16, 24, 32, 64, 128, 256]), "dtype": rng.choice(["f16", "bf16"]),
                 "gated": rng.random() < 0.5, "q_heads": kv_heads * rng.choice([1, 2, 3, 4, 4, 8]),
                 "kv_heads": kv_heads, "head_dim": head_dim}
            c["q_hi"] = _log_int(rng, 1, 2048)
            c["q_lo"] = rng.choice([1, c["q_hi"]])
            c["kv_hi"] = max(c["q_hi"], _log_int(rng, 1, 16384))
            c["kv_lo"] = rng.choice([min(c["q_hi"], c["kv_hi"]), c["kv_hi"]])
            if op == "prep":
                c["rotary"] = rng.choice([head_dim, head_dim // 4])
            tokens = c["batch"] * c["kv_hi"]
            scores = c["batch"] * c["q_heads"] * c["q_hi"] * c["kv_hi"]
            if tokens * c["kv_heads"] * c["head_dim"] > (1 << 27) or (op == "attend" and scores > (1 << 27)):
                continue
            if c["batch"] * c["q_hi"] * c["q_heads"] * c["head_dim"] > (1 << 23):
                continue
            return c
        if op == "span":
            c = {"op": op, "batch": _log_int(rng, 1, 64), "n_lo": 1, "n_hi": _log_int(rng, 1, 16),
                 "heads": rng.choice([4, 16]), "commit": rng.random() < 0.5}
            c["n_lo"] = rng.choice([1, c["n_hi"]])
            return c
        c = {"op": op, "batch": _log_int(rng, 1, 256), "rows_lo": 1, "rows_hi": rng.randint(1, 9),
             "vocab": _log_int(rng, 1000, 248320), "dtype": rng.choice(["f16", "bf16", "f32"]),
             "probs": rng.random() < 0.5, "greedy": rng.random() < 0.25}
        if c["batch"] * c["rows_hi"] * c["vocab"] <= 320 * 248320:
            return c


def _spread(n, lo, hi):
    """n whole numbers between lo and hi, the same for every seed, in no order."""
    return [lo + int((i * 0.6180339887498949 + 0.5) % 1.0 * (hi - lo + 1)) for i in range(n)]


def _lengths(case):
    q = _spread(case["batch"], case["q_lo"], case["q_hi"])
    kv = _spread(case["batch"], case["kv_lo"], case["kv_hi"])
    return q, [max(a, b) for a, b in zip(q, kv)]


def _starts(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def _span_lengths(case):
    n = _spread(case["batch"], case["n_lo"], case["n_hi"])
    take = [1 + i % m for i, m in enumerate(n)] if case["commit"] else n
    return n, take


def work(case):
    if case["op"] in ("attend", "prep"):
        q, kv = _lengths(case)
        hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
        if case["op"] == "attend":
            rows = sum(q) * hq * d * (3 if case["gated"] else 2)
            seen = sum(n * m - n * (n - 1) // 2 for n, m in zip(q, kv))
            return {"bytes": 2 * (rows + 2 * sum(kv) * hk * d), "flops": 4 * hq * d * seen}
        rows = sum(q) * d * 2 * (hq + 2 * hk)
        return {"bytes": 2 * rows + sum(q) * case["rotary"] * 4, "flops": 6 * rows}
    if case["op"] == "span":
        n, take = _span_lengths(case)
        b, h = case["batch"], case["heads"]
        state = b * h * 128 * 128 * 4 * (2 if case["commit"] else 1)
        conv = b * h * 384 * 4 * 2 * (2 if case["commit"] else 1)
        rows = sum(take) * h * 2 * ((256 if case["commit"] else 384) + 2 + (0 if case["commit"] else 256))
        return {"bytes": state + conv + rows, "flops": sum(take) * h * 128 * 128 * 4}
    rows = _spread(case["batch"], case["rows_lo"], case["rows_hi"])
    size = {"f16": 2, "bf16": 2, "f32": 4}[case["dtype"]]
    read = sum(rows) * case["vocab"] * size + (case["batch"] * case["vocab"] * 4 if case["probs"] else 0)
    return {"bytes": read + 8 * sum(rows), "flops": 3 * sum(rows) * case["vocab"]}


# ---- inputs -------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = {"device": "cuda", "generator": g}
    int32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")
    s = {"op": case["op"], "case": case}
    if case["op"] in ("attend", "prep"):
        dt, (q, kv) = DTYPES[case["dtype"]], _lengths(case)
        hq, hk, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
        need = [-(-n // page) for n in kv]
        width, pages, total = max(need), sum(need) + 3, sum(q)
        s["k_pages"] = torch.randn(pages, page, hk, d, dtype=dt, **dev)
        s["v_pages"] = torch.randn(pages, page, hk, d, dtype=dt, **dev)
        order = torch.randperm(pages, **dev).to(torch.int32)
        first = torch.tensor(_starts(need)[:-1], device="cuda")[:, None].long()
        s["page_table"] = order[(first + torch.arange(width, device="cuda")) % pages].contiguous()
        s["start"], s["kv_len"] = int32(_starts(q)), int32(kv)
        s["max_q"], s["max_kv"], s["total"] = max(q), max(kv), total
        if case["op"] == "attend":
            s["scale"] = 1.0 / math.sqrt(d)
            s["q"] = torch.randn(total, hq, d, dtype=dt, **dev)
            # the gate stays where the projection left it, beside the query of its head
            s["gate"] = torch.randn(total, hq, 2, d, dtype=dt, **dev)[:, :, 1] if case["gated"] else None
        else:
            s["rotary"], s["gated"] = case["rotary"], case["gated"]
            s["proj"] = torch.randn(total, (hq * (2 if case["gated"] else 1) + 2 * hk) * d, dtype=dt, **dev)
            s["q_norm"] = (torch.randn(d, **dev) * 0.1).to(dt)
            s["k_norm"] = (torch.randn(d, **dev) * 0.1).to(dt)
            freq = 1e7 ** (-np.arange(case["rotary"] // 2) * 2.0 / case["rotary"])
            ang = np.arange(max(kv))[:, None] * freq
            s["rope"] = torch.tensor(np.stack([np.cos(ang), np.sin(ang)], -1), dtype=torch.float32, device="cuda")
        return s
    if case["op"] == "span":
        n, take = _span_lengths(case)
        b, h, total = case["batch"], case["heads"], sum(n)
        half = lambda *shape, sd=1.0: (torch.randn(*shape, **dev) * sd).half()
        # one in-projection's rows: q, k, v, then the gate z, then a and b
        s["row"] = half(total, h * 512 + 2 * h)
        s["conv_weight"], s["conv_state"] = half(h * 384, 4, sd=0.5), half(b, h * 384, 4)
        s["state"] = torch.randn(b, h, 128, 128, **dev) * 0.05
        a_log = torch.rand(h, **dev) * 3 - 2
        s["a_log_bias"] = torch.stack([a_log, torch.randn(h, **dev) * 0.1], 1).contiguous()
        s["norm_weight"] = 1 + 0.1 * torch.randn(128, **dev)
        s["start"], s["max_n"] = int32(_starts(n)), max(take)
        s["counts"] = int32(take) if case["commit"] else None
        s["out"] = torch.zeros(total, h * 128, dtype=torch.float16, device="cuda")
        s["next_state"], s["next_conv"] = torch.empty_like(s["state"]), torch.empty_like(s["conv_state"])
        return s
    rows, v = _spread(case["batch"], case["rows_lo"], case["rows_hi"]), case["vocab"]
    total, starts = sum(rows), _starts(rows)
    s["start"], s["max_rows"] = int32(starts), max(rows)
    s["logits"] = (torch.randn(total, v, **dev) * 3).to(DTYPES[case["dtype"]])
    s["temperature"] = torch.zeros(case["batch"], device="cuda") if case["greedy"] \
        else 0.5 + torch.rand(case["batch"], **dev)
    s["u_accept"], s["u_sample"] = torch.rand(total, **dev), torch.rand(case["batch"], **dev)
    s["probs"] = None
    tokens = torch.randint(0, v, (total,), **dev)
    if case["probs"]:  # a draft model that is a little off, and tokens sampled from it
        heat = s["temperature"].clamp(min=0.5).repeat_interleave(torch.tensor(rows, device="cuda"))
        s["probs"] = torch.softmax((s["logits"].float() + 0.5 * torch.randn(total, v, **dev)) / heat[:, None], -1)
        drafted = torch.multinomial(s["probs"], 1, generator=g)[:, 0]
    else:  # a draft that is right three times in four
        best = s["logits"].float().argmax(-1)
        drafted = torch.where(torch.rand(total, **dev) < 0.75, best, torch.randint(0, v, (total,), **dev))
    tokens[1:] = drafted[:-1]
    s["tokens"] = tokens.to(torch.int32)
    return s


# ---- the operators, plain or the framework's ----------------------------------------------------------------------

def run(s):
    if own:
        import spock_b200
        return _own(spock_b200, s)
    return {"attend": _attend, "prep": _prep, "span": _span, "verify": _verify}[s["op"]](s)


def _own(lib, s):
    if s["op"] == "attend":
        return lib.paged_attention(s["q"], s["start"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_len"],
                                   s["scale"], gate=s["gate"])
    if s["op"] == "prep":
        q = lib.paged_attention_prep(s["proj"], s["start"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_len"],
                                     s["rope"], s["q_norm"], s["k_norm"], gated=s["gated"], eps=EPS)
        return q, s["k_pages"], s["v_pages"]
    if s["op"] == "span":
        h = s["state"].shape[1]
        layer = lib.DeltaNetLayer(s["conv_weight"], s["a_log_bias"], s["norm_weight"], num_heads=h, eps=EPS)
        qkv, z, a, b = s["row"].split([h * 384, h * 128, h, h], 1)
        if s["counts"] is None:
            return lib.deltanet_decode_span(layer, qkv, s["conv_state"], s["state"], a, b, z, s["start"],
                                            out=s["out"])
        lib.deltanet_decode_span(layer, qkv, s["conv_state"], s["state"], a, b, None, s["start"], counts=s["counts"],
                                 state_out=s["next_state"], conv_out=s["next_conv"])
        return s["next_state"], s["next_conv"]
    return lib.draft_verify(s["logits"], s["tokens"], s["start"], s["u_accept"], s["u_sample"], s["temperature"],
                            draft_probs=s["probs"])


def _rows(start, width, total):
    """[batch, width] row numbers of a padded form, which of them are real, and each row's place in that form."""
    at = start[:-1, None].long() + torch.arange(width, device=start.device)
    real = at < start[1:, None]
    seq = torch.searchsorted(start[1:].contiguous(), torch.arange(total, device=start.device, dtype=torch.int32),
                             right=True)
    return at.clamp(max=total - 1), real, seq, torch.arange(total, device=start.device) - start[:-1].long()[seq]


def _attend(s):
    q, start = s["q"], s["start"]
    total, hq, d = q.shape
    at, real, seq, place = _rows(start, s["max_q"], total)
    b, hk, m = at.shape[0], s["k_pages"].shape[2], s["max_kv"]
    k = s["k_pages"][s["page_table"].long()].reshape(b, -1, hk, d)[:, :m].float()
    v = s["v_pages"][s["page_table"].long()].reshape(b, -1, hk, d)[:, :m].float()
    rows = q[at].float().reshape(b, -1, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    score = (rows * s["scale"]) @ k.permute(0, 2, 3, 1)
    last = s["kv_len"][:, None] - (start[1:] - start[:-1])[:, None] + torch.arange(s["max_q"], device=q.device)
    seen = (torch.arange(m, device=q.device) <= last[:, :, None]) & real[:, :, None]
    seen = seen[:, None, None].expand(b, 1, hq // hk, s["max_q"], m).reshape(b, 1, -1, m)
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    norm = p.sum(-1, keepdim=True)
    o = (p @ v.transpose(1, 2)) / torch.where(norm == 0, 1.0, norm)
    o = o.reshape(b, hk, hq // hk, s["max_q"], d).permute(0, 3, 1, 2, 4).reshape(b, s["max_q"], hq, d)[seq, place]
    if s["gate"] is not None:
        o = o / (1 + torch.exp(-s["gate"].float()))
    return o.to(q.dtype)


def _turn(x, w, rope):
    """RMSNorm with (1 + w), then the rotation of the first dimensions."""
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1 + w)
    half = rope.shape[-2]
    c, n = rope[:, None, :, 0], rope[:, None, :, 1]
    lo, hi = y[..., :half], y[..., half:2 * half]
    return torch.cat([lo * c - hi * n, hi * c + lo * n, y[..., 2 * half:]], -1)


def _prep(s):
    proj, (pages, page, hk, d) = s["proj"], s["k_pages"].shape
    _, _, seq, place = _rows(s["start"], 1, s["total"])
    pos = (s["kv_len"] - (s["start"][1:] - s["start"][:-1])).long()[seq] + place
    x = proj.float().reshape(s["total"], -1, d)
    heads = x.shape[1] - 2 * hk
    q = x[:, :heads:2] if s["gated"] else x[:, :heads]
    rope = s["rope"][pos]
    to = (s["page_table"].long()[seq, pos // page], pos % page)
    s["k_pages"][to] = _turn(x[:, heads:heads + hk], s["k_norm"].float(), rope).to(proj.dtype)
    s["v_pages"][to] = proj.reshape(s["total"], -1, d)[:, heads + hk:]
    return _turn(q, s["q_norm"].float(), rope).to(proj.dtype), s["k_pages"], s["v_pages"]


def _span(s):
    start, h = s["start"], s["state"].shape[1]
    total, n = s["row"].shape[0], s["max_n"]
    at, real, seq, place = _rows(start, n, total)
    if s["counts"] is not None:
        real = real & (torch.arange(n, device=start.device) < s["counts"][:, None])
    qkv, z, a, b = s["row"].split([h * 384, h * 128, h, h], 1)
    x = torch.cat([s["conv_state"], qkv[at].transpose(1, 2)], 2)
    w = x.unfold(2, 4, 1)[:, :, 1:].float() * s["conv_weight"].float()[None, :, None]
    y = w.sum(-1)
    y = (y / (1 + torch.exp(-y))).reshape(at.shape[0], 3, h, 128, n)
    y = y.permute(4, 1, 0, 2, 3)
    q = y[:, 0] * torch.rsqrt((y[:, 0] ** 2).sum(-1, keepdim=True) + 1e-6) / math.sqrt(128)
    k = y[:, 1] * torch.rsqrt((y[:, 1] ** 2).sum(-1, keepdim=True) + 1e-6)
    v = y[:, 2]
    t = a[at].float() + s["a_log_bias"][:, 1]
    decay = torch.exp(-torch.exp(s["a_log_bias"][:, 0]) * (t.clamp(min=0) + torch.log1p(torch.exp(-t.abs()))))
    beta = 1 / (1 + torch.exp(-b[at].float()))
    state, outs = s["state"], []
    for i in range(n):
        new = state * decay[:, i, :, None, None]
        delta = beta[:, i, :, None] * (v[i] - (new * k[i][..., None]).sum(2))
        new = new + k[i][..., None] * delta[:, :, None]
        if s["counts"] is None:
            outs.append((new * q[i][..., None]).sum(2))
        state = torch.where(real[:, i, None, None, None], new, state)
    if s["counts"] is not None:
        window = s["counts"].long()[:, None, None] + torch.arange(4, device=start.device)
        s["next_conv"].copy_(torch.gather(x, 2, window.expand(-1, h * 384, 4)))
        s["next_state"].copy_(state)
        return s["next_state"], s["next_conv"]
    o = torch.stack(outs, 1)[seq, place]
    o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + EPS) * s["norm_weight"]
    gate = z.float().reshape(total, h, 128)
    s["out"].copy_((o * gate / (1 + torch.exp(-gate))).reshape(total, h * 128))
    return s["out"]


def _best(x):
    """The index of each row's largest value, the lowest among equals."""
    at = torch.arange(x.shape[-1], device=x.device)
    return torch.where(x == x.amax(-1, keepdim=True), at, x.shape[-1]).amin(-1)


def _verify(s):
    """In 64 bits: a sampled token is decided by which side of a border a sum falls on."""
    start, (total, vocab) = s["start"], s["logits"].shape
    at, real, seq, place = _rows(start, s["max_rows"], total)
    heat = s["temperature"].double()[seq]
    greedy = s["temperature"] == 0
    x = s["logits"].double() / torch.where(heat > 0, heat, 1.0)[:, None]
    best = _best(x)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    tested = torch.roll(s["tokens"], -1).long()[:, None]
    px = p.gather(1, tested)[:, 0]
    qx = s["probs"].gather(1, tested)[:, 0].double() if s["probs"] is not None else 1.0
    ok = torch.where(greedy[seq], best == tested[:, 0], s["u_accept"].double() * qx < px)
    ok = ok & (place < (start[1:] - start[:-1])[seq] - 1)
    taken = (ok[at] & real).long().cumprod(1).sum(1)
    row = start[:-1].long() + taken
    drafted = taken < (start[1:] - start[:-1]) - 1
    weight = p[row]
    if s["probs"] is not None:
        rest = (weight - s["probs"][row].double()).clamp(min=0)
    else:
        rest = weight.scatter(1, tested[row], 0.0)
    use = drafted & (rest.sum(-1) > 0)
    weight = torch.where(use[:, None], rest, weight)
    run_sum = weight.cumsum(-1)
    pick = (run_sum <= s["u_sample"].double()[:, None] * run_sum[:, -1:]).sum(-1).clamp(max=vocab - 1)
    pick = torch.where(greedy, best[row], pick)
    out = torch.where(place < taken[seq], tested[:, 0], torch.where(place == taken[seq], pick[seq], -1))
    return (taken + 1).to(torch.int32), out.to(torch.int32)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    start = s["start"].tolist()
    spans = list(zip(start[:-1], start[1:]))
    if case["op"] == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        group, page = case["q_heads"] // case["kv_heads"], case["page"]
        for b, (lo, hi) in enumerate(spans):
            length = int(s["kv_len"][b])
            where = torch.arange(length, device="cuda")
            ids = s["page_table"][b].long()[where // page]
            hidden = where[None] > (length - (hi - lo) + torch.arange(hi - lo, device="cuda"))[:, None]
            for h in range(case["q_heads"]):
                key, val = (t[ids, where % page, h // group].double() for t in (s["k_pages"], s["v_pages"]))
                score = s["q"][lo:hi, h].double() @ key.T * s["scale"]
                out[lo:hi, h] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ val
        return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())
    if case["op"] == "prep":
        k, v = s["k_pages"].double(), s["v_pages"].double()
        hq, hk, d, r = case["q_heads"], case["kv_heads"], case["head_dim"], case["rotary"]
        x = s["proj"].double().reshape(s["total"], -1, d)
        heads = x.shape[1] - 2 * hk
        pos = torch.cat([torch.arange(int(s["kv_len"][b]) - (hi - lo), int(s["kv_len"][b]), device="cuda")
                         for b, (lo, hi) in enumerate(spans)])
        turn = torch.view_as_complex(s["rope"].double())[pos][:, None]

        def normed(y, w):
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * (1 + w.double())
            z = torch.complex(y[..., :r // 2], y[..., r // 2:r]) * turn
            return torch.cat([z.real, z.imag, y[..., r:]], -1)

        q = normed(x[:, :heads].reshape(s["total"], hq, -1, d)[:, :, 0], s["q_norm"])
        new_k = normed(x[:, heads:heads + hk], s["k_norm"])
        for b, (lo, hi) in enumerate(spans):
            p = pos[lo:hi]
            ids = s["page_table"][b].long()[p // case["page"]]
            k[ids, p % case["page"]] = new_k[lo:hi]
            v[ids, p % case["page"]] = x[lo:hi, heads + hk:]
        return q, k, v
    if case["op"] == "span":
        h = case["heads"]
        qkv, z, a, bb = (t.double() for t in s["row"].split([h * 384, h * 128, h, h], 1))
        a_log, dt = s["a_log_bias"].double().unbind(1)
        out, states, convs = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda"), [], []
        for b, (lo, hi) in enumerate(spans):
            state, hist = s["state"][b].double(), s["conv_state"][b].double()
            n = hi - lo if s["counts"] is None else int(s["counts"][b])
            for t in range(lo, lo + n):
                hist = torch.cat([hist[:, 1:], qkv[t][:, None]], 1)
                y = (hist * s["conv_weight"].double()).sum(1)
                q, k, v = (y * torch.sigmoid(y)).reshape(3, h, 128)
                q = q / torch.sqrt(q.square().sum(-1, keepdim=True) + 1e-6)
                k = k / torch.sqrt(k.square().sum(-1, keepdim=True) + 1e-6)
                step = -torch.exp(a_log) * torch.nn.functional.softplus(a[t] + dt, threshold=1e9)
                state = state * torch.exp(step)[:, None, None]
                delta = torch.sigmoid(bb[t])[:, None] * (v - torch.einsum("hk,hkv->hv", k, state))
                state = state + torch.einsum("hk,hv->hkv", k, delta)
                if s["counts"] is None:
                    o = torch.einsum("hk,hkv->hv", q, state) / math.sqrt(128)
                    o = o / torch.sqrt(o.square().mean(-1, keepdim=True) + EPS) * s["norm_weight"].double()
                    g = z[t].reshape(h, 128)
                    out[t] = (o * g * torch.sigmoid(g)).reshape(-1)
            states.append(state)
            convs.append(hist)
        return out if s["counts"] is None else (torch.stack(states), torch.stack(convs))
    emitted, tokens = [], [-1] * start[-1]
    for b, (lo, hi) in enumerate(spans):
        heat, i = float(s["temperature"][b]), lo
        while True:
            x = s["logits"][i].double()
            p = None if heat == 0 else torch.softmax(x / heat, -1)
            if i == hi - 1:
                weight = p
                break
            t = int(s["tokens"][i + 1])
            if heat == 0:
                ok = int(torch.nonzero(x == x.max())[0]) == t
            else:
                qt = 1.0 if s["probs"] is None else float(s["probs"][i, t])
                ok = float(s["u_accept"][i]) * qt < float(p[t])
            if not ok:
                if heat != 0:
                    weight = p.clone()
                    if s["probs"] is None:
                        weight[t] = 0
                    else:
                        weight = (p - s["probs"][i].double()).clamp(min=0)
                    weight = weight if float(weight.sum()) > 0 else p
                break
            tokens[i] = t
            i += 1
        if heat == 0:
            tokens[i] = int(torch.nonzero(x == x.max())[0])
        else:
            c = weight.cumsum(0)
            tokens[i] = min(int((c <= float(s["u_sample"][b]) * c[-1]).sum()), case["vocab"] - 1)
        emitted.append(i - lo + 1)
    int32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    return int32(emitted), int32(tokens)
