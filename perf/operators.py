"""The mixer of a recurrent (gated delta rule) layer as measured cases: what a host that verifies drafts for a hybrid target runs
in those layers -- the prompt's short convolution, the chunked delta rule over the prompt, the few-row step of a verify or decode
pass, and the commit of the accepted rows into the state.

One head's state S (k_dim x v_dim, kept transposed: a row per value channel) goes from row to row as
    S <- e^g S;   u = beta (v - S^T k);   S <- S + k u^T;   o = scale S^T q
with q and k of unit length, g = -exp(a_log) softplus(a + dt_bias) <= 0 and beta = sigmoid(b); value head h reads key head
h // (v_heads / k_heads).  q, k and v come from a projection through a causal depthwise convolution and SiLU; the result is
normalised per head and gated with silu(z).  A verify pass has a tree of rows, every one continuing its parent's state.

The convolution's state is a ring of RING raw rows a sequence: position p lies in slot p % RING.  `base` is the position of a
sequence's first row; a sequence with base 0 starts from nothing, whatever its buffers hold."""
import math

import torch

own = False

RING = 32
CHUNK = 64
L2_EPS = 1e-6
NORM_EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TREE16 = [-1, 0, 0, 0, 0, 1, 5, 6, 2, 8, 9, 3, 11, 12, 4, 14]   # four children of the root, three chains of depth three, one extra leaf


def _case(what, heads, dims, dtype, lengths, name=None, **more):
    c = dict(what=what, k_heads=heads[0], v_heads=heads[1], k_dim=dims[0], v_dim=dims[1], taps=4, dtype=dtype,
             lengths=" ".join(str(n) for n in lengths), base=777, gated=True, tree=False, final=False, layers=1)
    c.update(more)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the next turn of a conversation on a small target: a few hundred rows behind a few thousand, not a multiple of anything
        _case("conv", (4, 8), (64, 64), "fp16", [299], "conv_followup_299", base=3001),
        # a document as prompt, the head counts of a mid-sized hybrid target
        _case("conv", (16, 32), (128, 128), "bf16", [8192], "conv_prompt_8192", base=0),
        # one row more than a block, few narrow heads: what the launches and one short walk cost
        _case("prefill", (4, 8), (64, 64), "fp16", [65], "prefill_short_65"),
        # the document again: one sequence, 32 heads, from an empty state
        _case("prefill", (16, 32), (128, 128), "bf16", [8192], "prefill_prompt_8192", base=0),
        # several conversations' prompts in one batch, from one row to a few thousand
        _case("prefill", (16, 32), (128, 128), "bf16", [1, 700, 64, 2049, 130, 1301], "prefill_ragged_6"),
        # a long document on an eighth of the heads, as one card of several holds them
        _case("prefill", (4, 8), (128, 128), "bf16", [32768], "prefill_long_32768", gated=False),
        # plain decoding: one row of one conversation, the new state written
        _case("step", (16, 32), (128, 128), "bf16", [1], "step_decode_1", final=True),
        # a verify pass of four proposals
        _case("step", (16, 32), (128, 128), "fp16", [5], "step_verify_5"),
        # tree drafts of four conversations
        _case("step", (16, 32), (128, 128), "bf16", [16] * 4, "step_tree_16x4", tree=True),
        # decoding 128 conversations at once
        _case("step", (16, 32), (128, 128), "bf16", [1] * 128, "step_decode_128", final=True),
        # the end of one conversation's round: three of five rows stay, in all of its recurrent layers
        _case("commit", (16, 32), (128, 128), "bf16", [5], "commit_5_24_layers", layers=24),
        # the end of a tree round of 32 conversations
        _case("commit", (16, 32), (128, 128), "bf16", [16] * 32, "commit_tree_16x32", tree=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    what = rng.choice(["conv", "prefill", "prefill", "step", "step", "commit"])
    k_heads = rng.choice([1, 2, 4, 8, 16])
    heads = (k_heads, k_heads * rng.choice([1, 2, 2, 3, 4] if k_heads < 16 else [1, 2]))
    dims = rng.choice([(64, 64), (64, 128), (128, 64), (128, 128), (128, 128), (128, 128)])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    more = dict(base=rng.choice([0, 1, 2, 31, _log(rng, 3, 60000)]), gated=rng.random() < 0.7)
    if what in ("conv", "prefill"):
        total = _log(rng, 1, 8192)
        n = rng.choice([1, 1, 1, 2, rng.randint(3, 12)])
        cuts = sorted(rng.randint(0, total) for _ in range(n - 1))
        lengths = [b - a for a, b in zip([0] + cuts, cuts + [total])]
        return _case(what, heads, dims, dtype, lengths, **more, taps=rng.choice([2, 3, 4, 4]))
    n = _log(rng, 1, 32)
    if what == "step":
        final, tree = rng.random() < 0.4, False
        if not final:
            tree = rng.random() < 0.5
        lengths = [rng.randint(1, 16) for _ in range(n)] if not final or rng.random() < 0.3 else [1] * n
        return _case(what, heads, dims, dtype, lengths, tree=tree, final=final, **more)
    return _case(what, heads, dims, dtype, [rng.randint(1, 16) for _ in range(n)], tree=rng.random() < 0.5,
                 layers=rng.randint(1, max(1, 24 // n)), **more)


# ---- what a program has in hand -------------------------------------------------------------------------------------------

def _lengths(c):
    """Rows of every sequence of the batch."""
    return [int(n) for n in c["lengths"].split()]


def _channels(c):
    return 2 * c["k_heads"] * c["k_dim"] + c["v_heads"] * c["v_dim"]


def _parents(case):
    """Parent of every row within its sequence, -1 for the first: a chain, or the branches of TREE16 cut to length."""
    return [p for n in _lengths(case) for p in (TREE16[:n] if case["tree"] else range(-1, n - 1))]


def _paths(case):
    """What an acceptance leaves for every sequence: the root path of one of its rows, as long ones as short ones."""
    out = []
    for s, n in enumerate(_lengths(case)):
        parent = TREE16[:n] if case["tree"] else list(range(-1, n - 1))
        at, path = (7 * s + 2) % n, []
        while at >= 0:
            path.append(at)
            at = parent[at]
        out.append(path[::-1])
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * int(seed) + 17)
    dt, dev = DTYPES[case["dtype"]], "cuda"
    hk, hv, dk, dv, n = case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"], len(_lengths(case))
    T, C, L = sum(_lengths(case)), _channels(case), case["layers"]
    randn = lambda *s: torch.randn(s, generator=gen, device=dev, dtype=torch.float32)  # noqa: E731
    rand = lambda *s: torch.rand(s, generator=gen, device=dev, dtype=torch.float32)  # noqa: E731
    offsets = [0]
    for length in _lengths(case):
        offsets.append(offsets[-1] + length)
    st = dict(case=case, offsets=offsets, off=torch.tensor(offsets, device=dev),
              base=torch.full((n,), case["base"], device=dev, dtype=torch.int64))
    # the decays of a trained layer: time constants from a few rows to a few thousand
    dt0 = torch.exp(rand(hv) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    st["a_log"] = torch.log(1.0 + 15.0 * rand(hv))
    st["dt_bias"] = dt0 + torch.log(-torch.expm1(-dt0))
    st["norm"] = 1.0 + 0.1 * randn(dv)
    st["conv"] = 0.5 * randn(C, case["taps"])
    if case["what"] in ("conv", "step"):
        st["qkv"], st["a"], st["b"] = randn(T, C).to(dt), randn(T, hv).to(dt), randn(T, hv).to(dt)
        st["ring"] = randn(n, RING, C).to(dt)
    if case["what"] == "conv":
        st["out"] = torch.empty((T, C), device=dev, dtype=dt)
        st["g"], st["beta"] = (torch.empty((T, hv), device=dev) for _ in range(2))
    if case["what"] == "prefill":
        # rows as the convolution leaves them: q and k of unit length with a part that all rows share, v behind SiLU
        unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # noqa: E731
        q, k = (unit(randn(T, hk, dk) + 0.5 * randn(1, hk, dk)).reshape(T, hk * dk) for _ in range(2))
        st["qkv"] = torch.cat([q, k, torch.nn.functional.silu(randn(T, hv * dv))], dim=1).to(dt)
        st["g"] = -torch.exp(st["a_log"]) * torch.nn.functional.softplus(randn(T, hv) + st["dt_bias"])
        st["beta"] = torch.sigmoid(randn(T, hv))
    if case["what"] in ("prefill", "step"):
        st["z"] = randn(T, hv * dv).to(dt)
        st["state"] = 0.1 * randn(n, hv, dv, dk)
        st["state_out"] = torch.empty_like(st["state"])
        st["out"] = torch.empty((T, hv * dv), device=dev, dtype=dt)
    if case["what"] == "step":
        st["parent"] = torch.tensor(_parents(case), device=dev, dtype=torch.int32)
        st["record"] = torch.empty((T * _record_row(case),), device=dev)
    if case["what"] == "commit":
        st["record"] = torch.stack([_pending(case, randn, rand) for _ in range(L)])
        st["state"] = 0.1 * randn(L, n, hv, dv, dk)
        st["state_out"] = torch.empty_like(st["state"])
        st["ring"] = randn(L, n, RING, C).to(dt)
        st["ring_before"] = st["ring"].clone()
        paths = _paths(case)
        st["keep"] = torch.tensor([len(p) for p in paths], device=dev)
        st["path"] = torch.tensor([p + [0] * (17 - len(p)) for p in paths], device=dev)
        st["results"] = _results(paths, case["base"])
    if own:
        _plan(st)
    torch.cuda.synchronize()
    return st


def _record_row(c):
    """f32 values that a verify pass leaves of a row: u of every value head, the unit k of every key head, its decays."""
    return c["v_heads"] * c["v_dim"] + c["k_heads"] * c["k_dim"] + c["v_heads"]


def _record_parts(c, record):
    T = sum(_lengths(c))
    a, b = T * c["v_heads"] * c["v_dim"], T * c["k_heads"] * c["k_dim"]
    return (record[..., :a].reshape(*record.shape[:-1], T, c["v_heads"], c["v_dim"]),
            record[..., a:a + b].reshape(*record.shape[:-1], T, c["k_heads"], c["k_dim"]),
            record[..., a + b:].reshape(*record.shape[:-1], T, c["v_heads"]))


def _pending(c, randn, rand):
    """A record as a verify pass leaves it."""
    T, hv, hk = sum(_lengths(c)), c["v_heads"], c["k_heads"]
    k = randn(T, hk, c["k_dim"])
    return torch.cat([0.5 * randn(T * hv * c["v_dim"]), (k / k.norm(dim=-1, keepdim=True)).reshape(-1), -0.3 * rand(T * hv)])


def _results(paths, base):
    """The acceptance's results as they lie in device memory: 112 bytes a sequence (accepted, committed, next, stopped, the draw
    counter, seventeen path entries and their number, the cursor, the margin)."""
    rows = torch.zeros((len(paths), 28), dtype=torch.int32)
    for s, p in enumerate(paths):
        rows[s, 0] = rows[s, 1] = len(p) - 1
        rows[s, 6:6 + len(p)] = torch.tensor(p, dtype=torch.int32)
        rows[s, 23] = len(p)
        rows[s, 24:26] = torch.tensor([base + len(p)]).view(torch.int32)
    return rows.cuda()


def _plan(st):
    """What a program that uses the library keeps beside its buffers: the layer's description, the batch's shape and where the
    buffers lie."""
    import turbospark_amd as ts
    c, kd = st["case"], st["case"]["k_heads"] * st["case"]["k_dim"]
    at = lambda k: st[k].data_ptr() if k in st else None  # noqa: E731
    st["layer"] = ts.GatedDelta(c["k_heads"], c["v_heads"], c["k_dim"], c["v_dim"], c["taps"], ts.BF16 if c["dtype"] == "bf16" else ts.F16,
                                conv=at("conv"), a_log=at("a_log"), dt_bias=at("dt_bias"), norm=at("norm"), l2_eps=L2_EPS, norm_eps=NORM_EPS)
    st["batch"] = st["layer"].batch(st["offsets"], at("base"), at("parent") if c["what"] == "step" and c["tree"] else None)
    gate = dict(z=at("z"), z_stride=st["z"].stride(0)) if "z" in st and c["gated"] else {}
    if c["what"] == "conv":
        # a pass is made again from the same position: it reads the ring as it was and writes a copy, or the last rows of 30 to 34 (and 62 to 66, ..)
        # would lie where the first ones' predecessors are read
        st["ring_before"], st["ring"] = st["ring"], st["ring"].clone()
        st["io"] = ts.GdnConv(qkv=at("qkv"), qkv_stride=st["qkv"].stride(0), a=at("a"), b=at("b"), gate_stride=st["a"].stride(0),
                              ring_in=at("ring_before"), ring_out=at("ring"), out=at("out"), out_stride=st["out"].stride(0), g=at("g"), beta=at("beta"))
    elif c["what"] == "prefill":
        st["workspace"] = torch.empty((st["layer"].prefill_workspace(st["batch"]),), device="cuda", dtype=torch.uint8)
        st["io"] = ts.GdnPrefill(q=at("qkv"), k=at("qkv") + 2 * kd, v=at("qkv") + 4 * kd, q_stride=st["qkv"].stride(0),
                                 k_stride=st["qkv"].stride(0), v_stride=st["qkv"].stride(0), g=at("g"), beta=at("beta"),
                                 state_in=at("state"), state_out=at("state_out"), out=at("out"), out_stride=st["out"].stride(0),
                                 workspace=at("workspace"), workspace_bytes=st["workspace"].numel(), **gate)
    elif c["what"] == "step":
        st["io"] = ts.GdnStep(qkv=at("qkv"), qkv_stride=st["qkv"].stride(0), a=at("a"), b=at("b"), gate_stride=st["a"].stride(0),
                              ring=at("ring"), state_in=at("state"), state_out=at("state_out") if c["final"] else None,
                              record=None if c["final"] else at("record"), out=at("out"), out_stride=st["out"].stride(0), **gate)
    else:
        st["io"] = ts.GdnCommit(n_layers=c["layers"], results=at("results"), record=at("record"), record_stride=4 * st["record"].stride(0),
                                ring_in=at("ring_before"), ring_out=at("ring"), ring_stride=st["ring"].stride(0), state_in=at("state"),
                                state_out=at("state_out"), state_stride=st["state"].stride(0))


# ---- one pass ---------------------------------------------------------------------------------------------------------------

def run(state):
    return (_own if own else _plain)[state["case"]["what"]](state)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_conv(st):
    st["layer"].conv(st["batch"], st["io"], _stream())
    return dict(rows=st["out"], g=st["g"], beta=st["beta"], ring=st["ring"])


def _own_prefill(st):
    st["layer"].prefill(st["batch"], st["io"], _stream())
    return dict(out=st["out"], state=st["state_out"])


def _own_step(st):
    st["layer"].step(st["batch"], st["io"], _stream())
    if st["case"]["final"]:
        return dict(out=st["out"], ring=st["ring"], state=st["state_out"])
    return dict(out=st["out"], ring=st["ring"], record=st["record"])


def _own_commit(st):
    st["layer"].commit(st["batch"], st["io"], _stream())
    return dict(ring=st["ring"], state=st["state_out"])


_own = dict(conv=_own_conv, prefill=_own_prefill, step=_own_step, commit=_own_commit)


# ---- the plain forms: elementary operations in 32 bits ------------------------------------------------------------------------

def _padded(off, T, M):
    """Row indices (sequences x M) of a ragged batch and which of them are rows; the others point at some row."""
    at = torch.arange(M, device=off.device)
    return (off[:-1, None] + at).clamp(max=T - 1), at < (off[1:] - off[:-1])[:, None]


def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _softplus(x):
    return x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


def _gate(st, o):
    """o in 32 bits, per head: the norm and the gate, then the one rounding."""
    c = st["case"]
    if c["gated"]:
        z = st["z"].float().reshape(o.shape)
        o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + NORM_EPS) * st["norm"] * _silu(z)
    return o.reshape(o.shape[0], -1).to(DTYPES[c["dtype"]])


def _conv_rows(st, parent, M):
    """The convolution's rows (sequences x M x channels, 32 bits, SiLU taken): tap j of a row is its j-th ancestor, and past the
    first row the ring's rows at positions base - 1, base - 2, ..  Returns them with the index table of the batch."""
    c, off, base = st["case"], st["off"], st["base"]
    idx, real = _padded(off, st["qkv"].shape[0], M)
    at = torch.arange(M, device=idx.device).expand(idx.shape)          # >= 0: a row of the pass; -1, -2, ..: position base - 1, base - 2, ..
    y = torch.zeros(*idx.shape, st["qkv"].shape[1], device=idx.device)
    seq = torch.arange(idx.shape[0], device=idx.device)[:, None]
    for j in range(c["taps"]):
        fresh = st["qkv"][(off[:-1, None] + at.clamp(min=0)).clamp(max=st["qkv"].shape[0] - 1)]
        kept = st["ring"][seq, (base[:, None] + at.clamp(max=-1)) % RING]
        x = torch.where((at >= 0)[..., None], fresh, kept).float() * (base[:, None] + at >= 0)[..., None]
        y += x * st["conv"][:, c["taps"] - 1 - j]
        if parent is None:
            at = at - 1
        else:
            at = torch.where(at >= 0, parent[(off[:-1, None] + at.clamp(min=0)).clamp(max=parent.numel() - 1)].long(), at - 1)
    return _silu(y), idx, real


def _heads(c, rows):
    kd = c["k_heads"] * c["k_dim"]
    q, k, v = rows[..., :kd], rows[..., kd:2 * kd], rows[..., 2 * kd:]
    shape = rows.shape[:-1]
    return (q.reshape(*shape, c["k_heads"], c["k_dim"]), k.reshape(*shape, c["k_heads"], c["k_dim"]),
            v.reshape(*shape, c["v_heads"], c["v_dim"]))


def _unit(x):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + L2_EPS)


def _gates(st):
    g = -torch.exp(st["a_log"]) * _softplus(st["a"].float() + st["dt_bias"])
    return g, 1.0 / (1.0 + torch.exp(-st["b"].float()))


def _ring_after(st, count):
    """The ring with the last `count` (at most) rows of every sequence in their slots."""
    off, base, ring = st["off"], st["base"], st["ring"].clone()
    n = off[1:] - off[:-1]
    at = n[:, None] - 1 - torch.arange(count, device=off.device)
    seq, which = (at >= 0).nonzero(as_tuple=True)
    row = at[seq, which]
    ring[seq, (base[seq] + row) % RING] = st["qkv"][off[seq] + row]
    return ring


def _plain_conv(st):
    c = st["case"]
    y, idx, real = _conv_rows(st, None, max(_lengths(c)))
    q, k, v = _heads(c, y[real])
    rows = torch.cat([_unit(q).flatten(1), _unit(k).flatten(1), v.flatten(1)], dim=1).to(DTYPES[c["dtype"]])
    g, beta = _gates(st)
    return dict(rows=rows, g=g, beta=beta, ring=_ring_after(st, c["taps"] - 1))


def _solve_rows(A):
    """(I + A)^-1 for strictly lower A, row by row: products of its powers, which would need no loop, cancel badly in 32 bits where
    keys are alike."""
    X = -A
    for i in range(1, A.shape[-1]):
        X[..., i, :i] += (X[..., i, :i, None] * X[..., :i, :i]).sum(-2)
    return X + torch.eye(A.shape[-1], device=A.device)


def _plain_prefill(st):
    c = st["case"]
    T, rep, scale = st["qkv"].shape[0], c["v_heads"] // c["k_heads"], c["k_dim"] ** -0.5
    N = -(-max(_lengths(c)) // CHUNK)
    idx, real = _padded(st["off"], T, N * CHUNK)
    x = st["qkv"][idx].float() * real[..., None]
    blocks = lambda t: t.unflatten(1, (N, CHUNK)).movedim(3, 1)  # noqa: E731  sequences x heads x blocks x CHUNK (x d)
    q, k, v = _heads(c, x)
    q, k, v = blocks(q).repeat_interleave(rep, 1), blocks(k).repeat_interleave(rep, 1), blocks(v)
    beta = blocks(st["beta"][idx] * real[..., None])
    G = blocks(st["g"][idx] * real[..., None]).double().cumsum(-1)        # differences of long sums: 64 bits
    low = torch.ones(CHUNK, CHUNK, device=x.device, dtype=torch.bool).tril()
    D = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~low, -math.inf)).float()
    kT = k.transpose(-1, -2)
    X = _solve_rows((beta[..., None] * D * (k @ kT)).tril(-1))
    eG = torch.exp(G).float()[..., None]
    U, W = X @ (beta[..., None] * v), X @ (beta[..., None] * eG * k)
    P, qd = D * (q @ kT), q * eG
    kd = (k * torch.exp(G[..., -1:] - G).float()[..., None]).transpose(-1, -2)
    end = eG[..., -1, :, None]
    S = (st["state"] * (st["base"] > 0)[:, None, None, None]).transpose(-1, -2)
    out = []
    for i in range(N):           # the recurrence itself
        u = U[:, :, i] - W[:, :, i] @ S
        out.append(qd[:, :, i] @ S + P[:, :, i] @ u)
        S = end[:, :, i] * S + kd[:, :, i] @ u
    o = scale * torch.stack(out, 2).flatten(2, 3).transpose(1, 2)[real]
    untouched = ((st["off"][1:] == st["off"][:-1]) & (st["base"] > 0))[:, None, None, None]
    return dict(out=_gate(st, o), state=torch.where(untouched, st["state"], S.transpose(-1, -2)).contiguous())


def _plain_step(st):
    c = st["case"]
    T, rep, scale, M = st["qkv"].shape[0], c["v_heads"] // c["k_heads"], c["k_dim"] ** -0.5, max(_lengths(c))
    y, idx, real = _conv_rows(st, st["parent"], M)
    q, k, v = _heads(c, y)
    q, k1 = _unit(q), _unit(k)
    q, k, v = q.transpose(1, 2).repeat_interleave(rep, 1), k1.transpose(1, 2).repeat_interleave(rep, 1), v.transpose(1, 2)
    g, beta = _gates(st)
    beta = (beta[idx] * real[..., None]).transpose(1, 2)
    # which rows lie on a row's root path, itself included
    row = torch.arange(M, device=idx.device)
    up = torch.where(real, st["parent"][idx].long(), -1)
    on = torch.zeros(*idx.shape, M, device=idx.device, dtype=torch.bool)
    at = row.expand(idx.shape)
    for _ in range(M):
        on |= (at[..., None] == row) & (at >= 0)[..., None]
        at = torch.where(at >= 0, up.gather(1, at.clamp(min=0)), at)
    G = torch.einsum("nij,njh->nhi", on.double(), (g[idx] * real[..., None]).double())
    on = on[:, None]
    D = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(~on, -math.inf)).float()
    S = st["state"] * (st["base"] > 0)[:, None, None, None]
    eG, ST = torch.exp(G).float()[..., None], S.transpose(-1, -2)
    X = _solve_rows((beta[..., None] * D * (k @ k.transpose(-1, -2))).tril(-1))
    u = X @ (beta[..., None] * (v - eG * (k @ ST)))
    o = scale * (eG * (q @ ST) + (D * (q @ k.transpose(-1, -2))) @ u)
    out, ring = _gate(st, o.transpose(1, 2)[real]), _ring_after(st, M)
    if c["final"]:
        last = (st["off"][1:] - st["off"][:-1] - 1)[:, None, None].expand(-1, c["v_heads"], 1)
        Gl = G.gather(2, last)
        w = torch.exp((Gl - G).masked_fill(~real[:, None], -math.inf)).float()
        state = torch.exp(Gl).float()[..., None] * S + (u * w[..., None]).transpose(-1, -2) @ k
        return dict(out=out, ring=ring, state=state)
    parts = (u.transpose(1, 2)[real], k1[real], g)
    return dict(out=out, ring=ring, record=torch.cat([p.reshape(-1) for p in parts]))


def _plain_commit(st):
    c, off, base, L = st["case"], st["off"], st["base"], st["case"]["layers"]
    u, k, g = _record_parts(c, st["record"])
    rep = c["v_heads"] // c["k_heads"]
    path, keep = st["path"], st["keep"]
    on = torch.arange(16, device=off.device) < keep[:, None]
    rows = off[:-1, None] + path[:, :16]
    u, k = u[:, rows], k[:, rows]                                          # layers x sequences x 16 x ..
    G = (g[:, rows] * on[:, :, None]).cumsum(2)
    end = G.gather(2, (keep - 1)[None, :, None, None].expand(L, -1, 1, c["v_heads"]))
    w = torch.exp(end - G) * on[:, :, None]
    S = st["state"] * (base > 0)[:, None, None, None]
    kept = (w[..., None] * u).permute(0, 1, 3, 4, 2) @ k.repeat_interleave(rep, 3).transpose(2, 3)
    ring = st["ring_before"].clone()
    seq, i = on.nonzero(as_tuple=True)
    ring[:, seq, (base[seq] + i) % RING] = st["ring_before"][:, seq, (base[seq] + path[seq, i]) % RING]
    return dict(ring=ring, state=torch.exp(end).squeeze(2)[..., None, None] * S + kept)


_plain = dict(conv=_plain_conv, prefill=_plain_prefill, step=_plain_step, commit=_plain_commit)


# ---- the operators' definition, row after row in 64 bits -----------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return dict(conv=_exact_conv, prefill=_exact_prefill, step=_exact_step, commit=_exact_commit)[case["what"]](st)


def _exact_convolved(st, s, parent):
    """Rows of one sequence behind the convolution and SiLU, gates beside them."""
    c, taps = st["case"], st["case"]["taps"]
    lo, hi, base = st["offsets"][s], st["offsets"][s + 1], int(st["base"][s])
    x = st["qkv"][lo:hi].double()
    before = torch.zeros(taps, x.shape[1], device=x.device, dtype=torch.float64)       # before[j]: position base - 1 - j
    for j in range(min(taps, base)):
        before[j] = st["ring"][s, (base - 1 - j) % RING].double()
    w = st["conv"].double()
    both = torch.cat([x, before])
    table = []
    for i in range(hi - lo):
        at, line = i, []
        for _ in range(taps):
            line.append(at if at >= 0 else hi - lo - at - 1)
            at = parent[at] if at >= 0 else at - 1
        table.append(line)
    table = torch.tensor(table, device=x.device, dtype=torch.int64).reshape(hi - lo, taps)
    y = sum(both[table[:, j]] * w[:, taps - 1 - j] for j in range(taps))
    y = y * torch.sigmoid(y)
    g = -torch.exp(st["a_log"].double()) * torch.logaddexp(st["a"][lo:hi].double() + st["dt_bias"].double(), torch.zeros((), device=x.device, dtype=torch.float64))
    q, k, v = _heads(c, y)
    q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + L2_EPS) for t in (q, k))
    return q, k, v, g, torch.sigmoid(st["b"][lo:hi].double())


def _exact_ring(st, count):
    ring = st["ring"].double()
    for s, n in enumerate(_lengths(st["case"])):
        for i in range(max(0, n - count), n):
            ring[s, (int(st["base"][s]) + i) % RING] = st["qkv"][st["offsets"][s] + i].double()
    return ring


def _exact_conv(st):
    parts = [_exact_convolved(st, s, range(-1, n - 1)) for s, n in enumerate(_lengths(st["case"]))]
    rows = torch.cat([torch.cat([t.flatten(1) for t in p[:3]], dim=1) for p in parts])
    return dict(rows=rows, g=torch.cat([p[3] for p in parts]), beta=torch.cat([p[4] for p in parts]), ring=_exact_ring(st, st["case"]["taps"] - 1))


def _exact_gate(st, o):
    if st["case"]["gated"]:
        z = st["z"].double().reshape(o.shape)
        o = o / torch.sqrt((o * o).mean(-1, keepdim=True) + NORM_EPS) * st["norm"].double() * z * torch.sigmoid(z)
    return o.reshape(o.shape[0], -1)


def _exact_row(c, S, q, k, v, g, beta):
    """One row through all heads of `S` (.. x heads x v_dim x k_dim)."""
    S = torch.exp(g)[..., None, None] * S
    u = beta[..., None] * (v - (S @ k[..., None]).squeeze(-1))
    S = S + u[..., None] * k[..., None, :]
    return S, u, c["k_dim"] ** -0.5 * (S @ q[..., None]).squeeze(-1)


def _exact_prefill(st):
    c = st["case"]
    rep = c["v_heads"] // c["k_heads"]
    q, k, v = (t.double() for t in _heads(c, st["qkv"]))
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    g, beta = st["g"].double(), st["beta"].double()
    S = st["state"].double() * (st["base"] > 0)[:, None, None, None]
    o = torch.zeros(q.shape[0], c["v_heads"], c["v_dim"], device=q.device, dtype=torch.float64)
    order = sorted(range(len(_lengths(c))), key=lambda s: -_lengths(c)[s])
    for i in range(max(_lengths(c))):
        live = [s for s in order if _lengths(c)[s] > i]
        if i == 0 or len(live) != at.numel():
            which = torch.tensor(live, device=q.device)
            at = torch.tensor([st["offsets"][s] for s in live], device=q.device)
        r = at + i
        S[which], _, o[r] = _exact_row(c, S[which], q[r], k[r], v[r], g[r], beta[r])
    for s, n in enumerate(_lengths(c)):
        if n == 0 and c["base"] > 0:
            S[s] = st["state"][s].double()
    return dict(out=_exact_gate(st, o), state=S)


def _exact_step(st):
    c = st["case"]
    rep = c["v_heads"] // c["k_heads"]
    out, us, ks, gs, ends = [], [], [], [], []
    parents = _parents(c)
    for s, n in enumerate(_lengths(c)):
        parent = parents[st["offsets"][s]:st["offsets"][s + 1]]
        q, k, v, g, beta = _exact_convolved(st, s, parent)
        root = st["state"][s].double() * (1.0 if c["base"] > 0 else 0.0)
        states = {-1: root}
        for i in range(n):
            states[i], u, o = _exact_row(c, states[parent[i]], q[i].repeat_interleave(rep, 0), k[i].repeat_interleave(rep, 0), v[i], g[i], beta[i])
            out.append(o)
            us.append(u)
        ks.append(k)
        gs.append(g)
        ends.append(states[n - 1])
    o, ring = _exact_gate(st, torch.stack(out)), _exact_ring(st, 16)
    if c["final"]:
        return dict(out=o, ring=ring, state=torch.stack(ends))
    return dict(out=o, ring=ring, record=torch.cat([torch.stack(us).reshape(-1), torch.cat(ks).reshape(-1), torch.cat(gs).reshape(-1)]))


def _exact_commit(st):
    c, L = st["case"], st["case"]["layers"]
    rep = c["v_heads"] // c["k_heads"]
    u, k, g = _record_parts(c, st["record"].double())
    ring, S = st["ring_before"].double(), st["state"].double()
    if c["base"] == 0:
        S = torch.zeros_like(S)
    for s, path in enumerate(_paths(c)):
        slots = ring[:, s].clone()
        for i, p in enumerate(path):
            r = st["offsets"][s] + p
            S[:, s] = torch.exp(g[:, r])[..., None, None] * S[:, s] + u[:, r][..., None] * k[:, r].repeat_interleave(rep, 1)[..., None, :]
            ring[:, s, (c["base"] + i) % RING] = slots[:, (c["base"] + p) % RING]
    return dict(ring=ring, state=S)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------

def work(case):
    hk, hv, dk, dv, n, T, C = (case["k_heads"], case["v_heads"], case["k_dim"], case["v_dim"], len(_lengths(case)), sum(_lengths(case)),
                               _channels(case))
    state, taps = 4.0 * hv * dk * dv, case["taps"]
    held = n if case["base"] > 0 else 0                                   # states that are read
    if case["what"] == "conv":
        return dict(bytes=4.0 * T * C + 12.0 * T * hv + 4.0 * C * taps + 4.0 * held * (taps - 1) * C, flops=T * C * (2.0 * taps + 6.0))
    if case["what"] == "prefill":
        row = 2.0 * C + 2.0 * hv * dv * (2 if case["gated"] else 1) + 8.0 * hv
        return dict(bytes=T * row + (n + held) * state, flops=6.0 * T * hv * dk * dv)
    if case["what"] == "step":
        row = 4.0 * C + 2.0 * hv * dv * (2 if case["gated"] else 1) + 4.0 * hv + (0.0 if case["final"] else 4.0 * _record_row(case))
        return dict(bytes=T * row + (held + (n if case["final"] else 0)) * state + 4.0 * C * taps, flops=T * (6.0 * hv * dk * dv + 2.0 * C * taps))
    kept = sum(len(p) for p in _paths(case))
    moved = sum(sum(i != p for i, p in enumerate(path)) for path in _paths(case)) * C * 4.0
    return dict(bytes=case["layers"] * ((n + held) * state + 4.0 * kept * _record_row(case) + moved), flops=case["layers"] * 2.0 * kept * hv * dk * dv)
