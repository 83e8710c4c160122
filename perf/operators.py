"""Operators of an 8-bit decoder layer that serves many adapters at once:

rows8     rows to e4m3 with a scale a row: behind the residual's addition and
          the RMS norm, behind silu(gate) * up, or as they are
linear8   the product of such rows with e4m3 weights of a scale a column
adapters  that product with the low-rank adapters of the rows' requests beside
          it: x A^T B^T of each row's own adapter

Run on the GPU. `own` chooses between elementary torch operations and the
framework's kernels; both take what prepare() makes.
"""
import torch

own = False

EPS = 1e-5
TOP = 448.0               # the largest e4m3 value
LEAST = 2.0 ** -100       # the least scale: rows of zeros have one too


def listed():
    return [
        # one row of a decode step of a model of 4096 channels
        {"name": "norm 1x4096", "op": "rows8", "source": "norm", "rows": 1,
         "width": 4096, "keep": False},
        # a long prompt of one of 5120, whose adapters read the bf16 rows too
        {"name": "norm 8192x5120", "op": "rows8", "source": "norm",
         "rows": 8192, "width": 5120, "keep": True},
        # a wide decode batch's attention result in front of its projection
        {"name": "plain 77x4096", "op": "rows8", "source": "plain", "rows": 77,
         "width": 4096, "keep": False},
        # a short prompt's feed-forward, in front of its second product
        {"name": "silu 509x14336", "op": "rows8", "source": "silu",
         "rows": 509, "width": 14336, "keep": False},
        # q, k and v of one decode row, with a bias
        {"name": "product 1x6144x4096", "op": "linear8", "rows": 1,
         "columns": 6144, "width": 4096, "bias": True},
        # gate and up of a decode batch
        {"name": "product 61x28672x4096", "op": "linear8", "rows": 61,
         "columns": 28672, "width": 4096, "bias": False},
        # the second product of a short prompt: few columns of long rows
        {"name": "product 523x4096x14336", "op": "linear8", "rows": 523,
         "columns": 4096, "width": 14336, "bias": False},
        # gate and up of a long prompt
        {"name": "product 8192x28672x4096", "op": "linear8", "rows": 8192,
         "columns": 28672, "width": 4096, "bias": False},
        # one request with an adapter, q, k and v
        {"name": "adapters 1x6144x4096", "op": "adapters", "rows": 1,
         "parts": "4096,1024,1024", "width": 4096, "slots": 4, "rank": 16,
         "mixed": False, "prompts": False},
        # a decode batch of as many adapters as half its rows, gate and up
        {"name": "adapters 64x28672x4096", "op": "adapters", "rows": 64,
         "parts": "14336,14336", "width": 4096, "slots": 32, "rank": 64,
         "mixed": True, "prompts": False},
        # prompts of several requests, q, k and v
        {"name": "adapters 2039x6144x4096", "op": "adapters", "rows": 2039,
         "parts": "4096,1024,1024", "width": 4096, "slots": 8, "rank": 32,
         "mixed": False, "prompts": True},
        # long prompts, the second product of the feed-forward
        {"name": "adapters 4097x4096x14336", "op": "adapters", "rows": 4097,
         "parts": "4096", "width": 14336, "slots": 8, "rank": 64,
         "mixed": True, "prompts": True},
    ]


def _spread(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    op = rng.choice(["rows8", "linear8", "linear8", "adapters", "adapters"])
    rows = _spread(rng, 1, 8192)
    if op == "rows8":
        source = rng.choice(["norm", "plain", "silu"])
        return {"op": op, "source": source, "rows": rows,
                "width": 8 * _spread(rng, 16, 1792 if source == "silu" else 1024),
                "keep": source == "norm" and rng.random() < .5}
    # widths and columns of the projections of layers, rarely a power of two
    width = 16 * _spread(rng, 32, 896)
    if op == "linear8":
        columns = 8 * _spread(rng, 64, 3584)
        while rows * columns * width > 8192 * 28672 * 4096:
            rows = (rows + 1) // 2
        return {"op": op, "rows": rows, "columns": columns, "width": width,
                "bias": rng.random() < .3}
    parts = [8 * _spread(rng, 32, 1792) for _ in range(rng.choice([1, 2, 3]))]
    slots = _spread(rng, 1, 48)
    rank = 8 * _spread(rng, 1, 16)
    while rows * (sum(parts) + slots * rank * len(parts)) * width > 4e11:
        rows = (rows + 1) // 2
    return {"op": op, "rows": rows, "parts": ",".join(map(str, parts)),
            "width": width, "slots": slots, "rank": rank,
            "mixed": rng.random() < .5, "prompts": rng.random() < .5}


def _parts(case):
    return [int(n) for n in case["parts"].split(",")]


def _weights(columns, width, gen):
    """e4m3 weights with a scale a column, as a checkpoint holds them."""
    w = torch.randn(columns, width, device="cuda", generator=gen) * width ** -.5
    scale = w.abs().amax(1).div_(TOP)
    return (w / scale[:, None]).to(torch.float8_e4m3fn), scale


def _activations(rows, width, gen):
    """bf16 rows of unlike lengths with some large channels, as a norm's are."""
    x = torch.randn(rows, width, device="cuda", generator=gen)
    x *= torch.exp(.5 * torch.randn(rows, 1, device="cuda", generator=gen))
    x *= torch.exp(.7 * torch.randn(width, device="cuda", generator=gen))
    return x.to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    T, K, op = case["rows"], case["width"], case["op"]
    if op == "rows8":
        state = {"op": op, "source": case["source"], "keep": case["keep"]}
        if case["source"] == "silu":
            state["x"] = (2 * torch.randn(T, 2 * K, device="cuda", generator=gen)
                          ).to(torch.bfloat16)
            return state
        state["x"] = _activations(T, K, gen)
        if case["source"] == "norm":
            state["residual"] = _activations(T, K, gen)
            state["weight"] = (1 + .1 * torch.randn(K, device="cuda", generator=gen)
                               ).to(torch.bfloat16)
        return state
    parts = _parts(case) if op == "adapters" else [case["columns"]]
    N = sum(parts)
    w, w_scale = _weights(N, K, gen)
    x = _activations(T, K, gen)
    q, scale = _eight(x.float())
    state = {"op": op, "q": q, "scale": scale, "w": w, "w_scale": w_scale,
             "bias": None}
    if op == "linear8":
        if case["bias"]:
            state["bias"] = torch.randn(N, device="cuda", generator=gen
                                        ).to(torch.bfloat16)
        return state
    S, R = case["slots"], case["rank"]
    state["x"] = x
    state["a"] = (torch.randn(S, len(parts) * R, K, device="cuda", generator=gen)
                  * K ** -.5).to(torch.bfloat16)
    state["b"] = (torch.randn(S, N, R, device="cuda", generator=gen)
                  * .5 * R ** -.5).to(torch.bfloat16)
    ranks = torch.randint(1, R + 1, (S,), generator=host) if case["mixed"] \
        else torch.full((S,), R)
    # every eighth request, about, has no adapter: slot -1
    if case["prompts"]:
        cuts = torch.randint(0, T + 1, (2 * S - 1,), generator=host).sort().values
        seq = torch.bucketize(torch.arange(T), cuts, right=True)
        of = torch.randint(0, S, (2 * S,), generator=host)
        none = torch.rand(2 * S, generator=host) < .125
        slots = torch.where(none, -1, of)[seq]
    else:
        slots = torch.randint(0, S, (T,), generator=host)
        if T > 1:
            slots[torch.rand(T, generator=host) < .125] = -1
    # the rows adapter by adapter, those without one at the end
    key = torch.where(slots < 0, S, slots)
    state["order"] = key.argsort(stable=True).to(torch.int32).cuda()
    state["starts"] = torch.searchsorted(
        key.sort().values, torch.arange(S + 1)).to(torch.int32).cuda()
    state["slots"] = slots.cuda()
    state["ranks"] = ranks.to(torch.int32).cuda()
    state["ends"] = tuple(torch.tensor(parts).cumsum(0).tolist())
    return state


def _eight(v):
    """Rows as e4m3 values and a scale each: the largest one becomes 448."""
    scale = (v.abs().amax(1) / TOP).clamp(min=LEAST)
    return (v / scale[:, None]).to(torch.float8_e4m3fn), scale


def _source(state, real):
    """The rows that become 8 bits, and what else the pass returns."""
    x = state["x"].to(real)
    if state["source"] == "silu":
        g, u = x.chunk(2, 1)
        return g / (1 + torch.exp(-g)) * u, {}
    if state["source"] == "plain":
        return x, {}
    total = (x + state["residual"].to(real)).to(torch.bfloat16)
    t = total.to(real)
    rows = t / torch.sqrt(t.square().mean(1, keepdim=True) + EPS) \
        * state["weight"].to(real)
    return rows, {"residual": total} | ({"rows": rows} if state["keep"] else {})


def _low_rank(state, real):
    """x A^T B^T, of every adapter, with the others' middle values as zeros."""
    x, a, b = (state[k].to(real) for k in ("x", "a", "b"))
    S, N, R = b.shape
    ends, count = state["ends"], len(state["ends"])
    middle = (x @ a.reshape(-1, a.shape[2]).T).view(-1, S, count, R)
    at = torch.arange(S, device=x.device)
    mine = state["slots"][:, None] == at
    held = torch.arange(R, device=x.device) < state["ranks"][:, None]
    middle = torch.where((mine[:, :, None] & held)[:, :, None], middle, 0)
    return torch.cat([
        middle[:, :, p].reshape(-1, S * R)
        @ b[:, first:end].transpose(1, 2).reshape(S * R, end - first)
        for p, (first, end) in enumerate(zip((0,) + ends, ends))], 1)


def _product(state, real):
    y = state["q"].to(real) @ state["w"].to(real).T
    y = y * state["scale"].to(real)[:, None] * state["w_scale"].to(real)
    return y if state["bias"] is None else y + state["bias"].to(real)


def run(state):
    op = state["op"]
    if own:
        from gpustack_amd import ops

        if op == "rows8":
            more = {}
            if state["source"] == "norm":
                r, more["residual"] = ops.add_rms_norm_fp8(
                    state["x"], state["residual"], state["weight"], EPS,
                    rows=state["keep"])
                if state["keep"]:
                    more["rows"] = r.rows
            elif state["source"] == "silu":
                r = ops.silu_and_mul_fp8(state["x"])
            else:
                r = ops.rows_fp8(state["x"])
            return {"q": r.q, "scale": r.scale} | more
        y = ops.linear_fp8(state["q"], state["scale"], state["w"],
                           state["w_scale"], state["bias"])
        if op == "adapters":
            ops.lora_add(y, state["x"], state["a"], state["b"], state["order"],
                         state["starts"], state["ranks"], state["ends"])
        return y
    if op == "rows8":
        rows, more = _source(state, torch.float32)
        q, scale = _eight(rows)
        if "rows" in more:
            more["rows"] = rows.to(torch.bfloat16)
        return {"q": q, "scale": scale} | more
    y = _product(state, torch.float32)
    if op == "adapters":
        y = y + _low_rank(state, torch.float32)
    return y.to(torch.bfloat16)


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point()
         else v for k, v in s.items()}
    if case["op"] == "rows8":
        x = d["x"]
        out = {}
        if case["source"] == "silu":
            half = x.shape[1] // 2
            rows = x[:, :half] * torch.sigmoid(x[:, :half]) * x[:, half:]
        elif case["source"] == "plain":
            rows = x
        else:
            # the sum is held in bf16, and that is what is normed
            out["residual"] = (x + d["residual"]).to(torch.bfloat16).double()
            length = (out["residual"] ** 2).sum(1, keepdim=True) / x.shape[1]
            rows = out["residual"] * (length + EPS) ** -.5 * d["weight"]
            if case["keep"]:
                out["rows"] = rows
        out["scale"] = torch.maximum(rows.abs().max(1).values / TOP,
                                     torch.tensor(LEAST, device=x.device).double())
        out["q"] = (rows / out["scale"][:, None]).to(torch.float8_e4m3fn).double()
        return out
    y = torch.nn.functional.linear(d["q"] * d["scale"][:, None],
                                   d["w"] * d["w_scale"][:, None], d["bias"])
    if case["op"] == "adapters":
        R, ends = case["rank"], d["ends"]
        for slot in range(case["slots"]):
            rows = (s["slots"] == slot).nonzero()[:, 0]
            r = int(s["ranks"][slot])
            first = 0
            for p, end in enumerate(ends):
                down = d["a"][slot, p * R:p * R + r]
                up = d["b"][slot, first:end, :r]
                y[rows, first:end] += d["x"][rows] @ down.T @ up.T
                first = end
    return y


def work(case):
    T, K = case["rows"], case["width"]
    if case["op"] == "rows8":
        many = {"plain": 2, "silu": 4, "norm": 6}[case["source"]] \
            + (2 if case["keep"] else 0)
        return {"bytes": T * K * (many + 1) + 4 * T
                + (2 * K if case["source"] == "norm" else 0),
                "flops": T * K * {"plain": 2, "silu": 6, "norm": 7}[case["source"]]}
    parts = _parts(case) if case["op"] == "adapters" else [case["columns"]]
    N = sum(parts)
    moved = T * K + N * K + 4 * (T + N) + 2 * T * N
    flops = 2 * T * N * K
    if case["op"] == "linear8":
        return {"bytes": moved + (2 * N if case["bias"] else 0), "flops": flops}
    rank = (case["rank"] + 1) / 2 if case["mixed"] else case["rank"]
    # rows on average with an adapter, and adapters that have a row
    rows = T if T == 1 else T * 7 / 8
    used = case["slots"] * (1 - (1 - 1 / case["slots"])
                            ** (2 * case["slots"] if case["prompts"] else rows))
    used = min(max(used, 1), T)
    return {"bytes": int(moved + 2 * rows * K
                         + 2 * used * rank * (len(parts) * K + N)),
            "flops": int(flops + 2 * rows * rank * (len(parts) * K + N))}
