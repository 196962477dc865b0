"""The engine with low-rank adapters per sequence (laya_forward_adapted): against
an engine whose weights have the adapter merged in, against a layer in 32-bit
PyTorch, and the operators run one after another as that layer does.

Adapter matrices: A about 1/sqrt(in), B about 0.02, scale 2, so the adapter's
part of a projection is a fifth to a half of the projection itself.
"""
import os

import numpy as np
import pytest
import torch

from laya_rust_b200 import arch, gguf, modelgen, ops
from laya_rust_b200 import engine as E
from test_gpu_parity import synthetic_req

pytestmark = pytest.mark.gpu

PROJ = (arch.wqkv, arch.wo_attn, arch.wi, arch.wo_mlp)
RANKS = {0: 16, 1: 5, 2: 40}
SCALE = {0: 2.0, 1: -1.5, 2: 0.75}


def matrices(slot, name):
    out, inn = arch.stored_shapes()[name]
    g = np.random.default_rng([slot, sum(name.encode())])
    a = (g.standard_normal((RANKS[slot], inn)) * inn ** -0.5).astype(np.float16)
    b = (g.standard_normal((out, RANKS[slot])) * 0.02).astype(np.float16)
    return a, b


def names(slot):
    """Slot 0 adapts everything, 1 the attention of odd layers, 2 the FFN."""
    for i in range(arch.NLAYER):
        for p in PROJ:
            if slot == 0 or (slot == 1 and i % 2 and p in PROJ[:2]) or (slot == 2 and p in PROJ[2:]):
                yield p(i)


def install(eng):
    eng.adapters_create(4, 48)
    for s in RANKS:
        eng.adapter_create(s, RANKS[s], SCALE[s])
        for n in names(s):
            eng.adapter_upload(s, n, *matrices(s, n))


@pytest.fixture(scope="module")
def header():
    return gguf.read(modelgen.cached_model(seed=0))


@pytest.fixture(scope="module")
def engine():
    e = E.Engine(modelgen.cached_model(seed=0), device=0)
    install(e)
    yield e
    e.close()


def weight(header, name):
    return header.f32(name).reshape(arch.stored_shapes()[name])


@pytest.fixture(scope="module")
def merged(header):
    """One engine per slot, its weights W + scale B A."""
    made = {}

    def get(slot):
        if slot not in made:
            e = E.Engine(modelgen.cached_model(seed=0), device=0)
            for n in names(slot):
                a, b = (v.astype(np.float32) for v in matrices(slot, n))
                e.upload_f32(n, weight(header, n) + SCALE[slot] * (b @ a))
            made[slot] = e
        return made[slot]

    yield get
    for e in made.values():
        e.close()


def on(req):
    return req.mmask.reshape(req.n, req.k) != 0


# a single request (split K), one row block, several, sequences of the flash
# kernel, and 900 rows, whose Wi leaves a partial round of tiles (run as halves)
LENS = [[90, 89], [31, 77, 128, 64, 90, 12, 1 + 4], [300, 40, 400, 128, 129, 77, 256, 200, 30, 390, 64, 100],
        [60 + (7 * i) % 69 for i in range(128)], [100] * 9]
IDS = ["request", "one-block", "long", "batch", "halves"]


@pytest.mark.parametrize("lens", LENS, ids=IDS)
def test_against_merged_weights(engine, merged, lens):
    """Every sequence under one adapter equals the engine whose weights hold
    it, within the parity bar the engine has against the reference's f32
    backend (2e-2 + 1e-2 |want|: the merged weights are rounded to f16 anew)."""
    req = synthetic_req(3, lens, 4)
    base = engine.forward(req)
    for slot in RANKS:
        got = engine.forward(req, adapters=[slot] * req.n)
        want = merged(slot).forward(req)
        for g, w in ((got.logits, want.logits), (got.act, want.act)):
            err = np.abs(g - w)
            assert np.all(np.isfinite(g)) and err.max() <= 2e-2 and np.all(err <= 2e-2 + 1e-2 * np.abs(w)), float(err.max())
        m = on(req).ravel()
        moved = np.abs(want.logits - base.logits)[m].max()
        assert moved > 4 * np.abs(got.logits - want.logits)[m].max(), moved   # the adapter is what the answers follow


@pytest.mark.parametrize("lens", LENS, ids=IDS)
def test_sequences_keep_to_their_own_adapter(engine, lens):
    """A mixed batch: each sequence bit for bit as in a batch where all have
    its adapter (adapters of other rows add exact zeros), and those without one
    as in laya_forward."""
    req = synthetic_req(4, lens, 4)
    who = np.array([(i % 4) - 1 for i in range(req.n)])
    got = engine.forward(req, adapters=who)
    for slot in (-1, 0, 1, 2):
        alone = engine.forward(req) if slot < 0 else engine.forward(req, adapters=[slot] * req.n)
        for b in np.flatnonzero(who == slot):
            assert np.array_equal(got.logits.reshape(req.n, -1)[b], alone.logits.reshape(req.n, -1)[b]), (slot, b)
            assert np.array_equal(got.act.reshape(req.n, 2)[b], alone.act.reshape(req.n, 2)[b]), (slot, b)


def test_no_adapters_is_the_plain_forward(engine):
    req = synthetic_req(5, [200, 33, 64], 3)
    a, b = engine.forward(req), engine.forward(req, adapters=[-1, -1, -1])
    assert np.array_equal(a.logits, b.logits) and np.array_equal(a.act, b.act)


def test_graph_replays_and_other_assignments(engine):
    """Eager, captured and replayed calls agree bit for bit; another assignment
    and another request of the same shape reach the launches."""
    req = synthetic_req(6, [120, 100, 90, 80], 4)
    first = engine.forward(req, adapters=[0, 1, -1, 2])
    for _ in range(3):
        again = engine.forward(req, adapters=[0, 1, -1, 2])
        assert np.array_equal(first.logits, again.logits) and np.array_equal(first.act, again.act)
    # the same set of slots in the same order of first use, other rows
    r2 = synthetic_req(7, [120, 100, 90, 80], 4)
    assert not np.array_equal(r2.ids, req.ids)
    got = engine.forward(r2, adapters=[0, 1, -1, 2])
    plan = engine.plan(r2, adapters=[0, 1, -1, 2])
    plan.run()
    want = plan.outputs()
    assert np.array_equal(got.logits, want.logits)
    swapped = engine.forward(req, adapters=[1, 0, 2, -1])
    assert not np.array_equal(swapped.logits, first.logits)
    plan.capture()
    for _ in range(2):
        plan.run()
        out = plan.outputs()
        assert np.array_equal(out.logits, want.logits) and np.array_equal(out.act, want.act)
    plan.close()


def test_uploads_reach_the_next_call_and_drops_are_refused():
    eng = E.Engine(modelgen.cached_model(seed=0), device=0)
    try:
        req = synthetic_req(8, [64, 50], 3)
        base = eng.forward(req)
        eng.adapters_create(2, 32)
        with pytest.raises(E.LayaError, match="not a created slot") as ei:
            eng.forward(req, adapters=[0, -1])
        assert ei.value.code == E.LAYA_E_INVALID
        eng.adapter_create(0, 8, 1.0)
        outs = [eng.forward(req, adapters=[0, -1]) for _ in range(3)]
        # a slot without matrices changes nothing
        assert all(np.array_equal(o.logits, base.logits) for o in outs)
        n = arch.wqkv(3)
        out, inn = arch.stored_shapes()[n]
        g = np.random.default_rng(0)
        a, b = (g.standard_normal((8, inn)) * 0.03).astype(np.float32), (g.standard_normal((out, 8)) * 0.1).astype(np.float32)
        eng.adapter_upload(0, n, a, b)
        one = eng.forward(req, adapters=[0, -1])
        k = req.k
        assert not np.array_equal(one.logits[:k], base.logits[:k]) and np.array_equal(one.logits[k:], base.logits[k:])
        plan = eng.plan(req, adapters=[0, -1])
        plan.capture()
        eng.adapter_upload(0, n, a, 2 * b)
        plan.run()
        two = plan.outputs()
        assert np.array_equal(two.logits, eng.forward(req, adapters=[0, -1]).logits)
        assert not np.array_equal(two.logits, one.logits)
        eng.adapter_create(0, 20, 1.0)                    # two chunks: the plan is stale
        for f in (plan.run, plan.capture, lambda: plan.run_layer(0), lambda: plan.profile(1)):
            with pytest.raises(E.LayaError, match="dropped or changed its rank") as ei:
                f()
            assert ei.value.code == E.LAYA_E_STATE
        assert np.array_equal(eng.forward(req, adapters=[0, -1]).logits, base.logits)   # created anew: empty
        eng.adapter_drop(0)
        for f in (lambda: eng.forward(req, adapters=[0, -1]), lambda: eng.plan(req, adapters=[0, -1]),
                  lambda: eng.forward(req, adapters=[2, -1]), lambda: eng.forward(req, adapters=[-2, -1])):
            with pytest.raises(E.LayaError, match="not a created slot"):
                f()
        eng.adapters_create(1, 16)
        with pytest.raises(E.LayaError) as ei:
            plan.run()
        assert ei.value.code == E.LAYA_E_STATE
        plan.close()
        assert np.array_equal(eng.forward(req).logits, base.logits)
        L = E.lib()
        for rc in (L.laya_adapters_create(eng._h, 0, 16), L.laya_adapters_create(eng._h, 4097, 16),
                   L.laya_adapters_create(eng._h, 1, 257), L.laya_adapter_create(eng._h, 1, 4, 1.0),
                   L.laya_adapter_create(eng._h, 0, 17, 1.0), L.laya_adapter_create(eng._h, 0, 0, 1.0),
                   L.laya_adapter_create(eng._h, 0, 4, float("inf")), L.laya_adapter_drop(eng._h, -1)):
            assert rc == E.LAYA_E_INVALID
        with pytest.raises(E.LayaError) as ei:
            eng.adapter_upload(0, n, a[:4], b[:, :4])
        assert ei.value.code == E.LAYA_E_STATE             # the slot is empty
        eng.adapter_create(0, 4, 1.0)
        with pytest.raises(E.LayaError, match="not an encoder projection"):
            eng.adapter_upload(0, "scorer.1.weight", np.zeros((4, 1024)), np.zeros((1024, 4)))
        with pytest.raises(E.LayaError, match="not finite"):
            eng.adapter_upload(0, n, a[:4] * np.nan, b[:, :4])
        with pytest.raises(E.LayaError, match="not finite"):
            eng.adapter_upload(0, n, a[:4], b[:, :4] * 1e7)
        assert np.array_equal(eng.forward(req, adapters=[0, 0]).logits, base.logits)   # nothing was taken
    finally:
        eng.close()


def test_requests_of_several_tenants_share_forwards(engine, merged):
    """Request JSON to response JSON, each request under its own adapter, packed
    together: the answers of the engine whose weights hold that adapter, within
    the front end's bar (2e-2 on probabilities)."""
    from laya_rust_b200 import frontend as FE, tokgen, workloads
    words = workloads.vocab_words(tokgen.tokenizer_json(0))
    reqs = [workloads.single_request_json(words, i) for i in range(5)]
    who = [0, -1, 2, 1, 0]
    tok = FE.Tokenizer(gguf_path=modelgen.cached_model(seed=0))
    got = FE.run_requests(engine, tok, reqs, across_requests=True, adapters=who)
    base = FE.run_requests(engine, tok, reqs, across_requests=True)
    moved = 0.0
    for i, slot in enumerate(who):
        want = FE.run_requests(engine if slot < 0 else merged(slot), tok, [reqs[i]])[0]
        assert set(got[i]["answers"]) == set(want["answers"])
        for qid, w in want["answers"].items():
            g, b = got[i]["answers"][qid], base[i]["answers"][qid]
            for k, p in w.get("probabilities", {}).items():
                assert abs(g["probabilities"][k] - p) <= 2e-2
                moved = max(moved, abs(b["probabilities"][k] - p))
            assert abs(g["rl_agent"]["act_probability"] - w["rl_agent"]["act_probability"]) <= 2e-2
    assert moved > 1e-3
    with pytest.raises(ValueError):
        FE.run_requests(engine, tok, reqs, adapters=[0])
    tok.close()


def test_an_engine_without_weights_refuses():
    eng = E.Engine(None, device=0)
    try:
        with pytest.raises(E.LayaError) as ei:
            eng.adapters_create(1, 16)
        assert ei.value.code == E.LAYA_E_STATE
        with pytest.raises(E.LayaError) as ei:
            ops.set_rope_scaling(eng)
        assert ei.value.code == E.LAYA_E_STATE
    finally:
        eng.close()


# ---- one layer against PyTorch, and the operators in its place -------------------
def torch_layer(header, layer, x, lens, who, freqs, m):
    """The encoder layer in 32 bits (x [R, 1024] on the GPU), each sequence with
    its adapter merged, frequencies `freqs` and factor m."""
    dev = x.device

    def proj(h, name, slot):
        y = h @ torch.from_numpy(weight(header, name)).to(dev).T
        if slot >= 0 and name in set(names(slot)):
            a, b = (torch.from_numpy(v.astype(np.float32)).to(dev) for v in matrices(slot, name))
            y = y + SCALE[slot] * ((h @ a.T) @ b.T)
        return y

    def norm(h, name):
        w = torch.from_numpy(header.f32(name)).to(dev)
        return torch.nn.functional.layer_norm(h, (1024,), w, None, arch.EPS)

    out, row = [], 0
    for ln, slot in zip(lens, who):
        h = x[row:row + ln]
        row += ln
        qkv = proj(norm(h, arch.attn_norm(layer)), arch.wqkv(layer), slot).view(ln, 3, 16, 64)
        ang = torch.arange(ln, device=dev, dtype=torch.float64)[:, None] * torch.from_numpy(freqs).to(dev)[None]
        c, s = (m * ang.cos()).float()[:, None], (m * ang.sin()).float()[:, None]
        rot = lambda t: torch.cat([t[..., :32] * c - t[..., 32:] * s, t[..., 32:] * c + t[..., :32] * s], -1) * arch.SCALE
        q, k, v = rot(qkv[:, 0]), rot(qkv[:, 1]), qkv[:, 2]
        sc = torch.einsum("qhd,khd->hqk", q, k)
        if layer % 3:
            i = torch.arange(ln, device=dev)
            sc = sc.masked_fill((i[:, None] - i[None]).abs() > arch.WINDOW, float("-inf"))
        ctx = torch.einsum("hqk,khd->qhd", sc.softmax(-1), v).reshape(ln, 1024)
        h = h + proj(ctx, arch.wo_attn(layer), slot)
        g = proj(norm(h, f"encoder.layers.{layer}.mlp_norm.weight"), arch.wi(layer), slot)
        h = h + proj(torch.nn.functional.gelu(g[:, :2624]) * g[:, 2624:], arch.wo_mlp(layer), slot)
        out.append(h)
    return torch.cat(out)


@pytest.mark.parametrize("lens", [[90, 89], [300, 40, 200, 128, 129, 77], [60 + (7 * i) % 69 for i in range(64)], [100] * 9,
                                  [1500, 40, 700]],
                         ids=["request", "long", "batch", "halves", "beyond-512"])
@pytest.mark.parametrize("layer", [1, 3])
def test_a_layer_with_mixed_adapters_and_stretched_rotation(engine, header, lens, layer):
    """Relative error under 1e-2 per row, the bar of the plain layer's test."""
    req = synthetic_req(9, lens, 2)
    who = [(i % 4) - 1 for i in range(len(lens))]
    x = np.random.default_rng(2).standard_normal((sum(lens), 1024)).astype(np.float32)
    sc = ops.RopeScaling(ops.ROPE_PARTS, 4.0, 128.0, 1.0, 16.0)
    theta = modelgen.THETA_SLIDING if layer % 3 else modelgen.THETA_FULL
    freqs, m = ops.rope_freqs(theta, 64, sc)
    plan = engine.plan(req, adapters=who)
    try:
        ops.set_rope_scaling(engine, sc, sc)
        plan.set_hidden(x)
        plan.run_layer(layer)
        got = torch.from_numpy(plan.hidden())
    finally:
        ops.set_rope_scaling(engine)
        plan.close()
    want = torch_layer(header, layer, torch.from_numpy(x).cuda(), lens, who, freqs, m).cpu()
    plain = torch_layer(header, layer, torch.from_numpy(x).cuda(), lens, [-1] * len(lens), freqs, m).cpu()
    rel = (got - want).norm(dim=1) / want.norm(dim=1)
    assert float(rel.max()) < 1e-2, float(rel.max())
    has = torch.repeat_interleave(torch.tensor(who), torch.tensor(lens))
    # a wrong or missing adapter would show: it moves those rows by far more
    moved = (plain - want).norm(dim=1) / want.norm(dim=1)
    strong = (has == 0) | (has == 2)
    assert float(moved[strong].min()) > 10 * float(rel.max())


def test_projection_rotation_and_attention_one_after_another(header):
    """laya_lora_run into a q|k|v buffer, laya_rope on its q and k in place (the
    factor on cos and sin carries the attention scale), then the engine's
    attention kernel; against 64 bits.

    Tolerance: q and k are rounded to f16 twice, the attention scale between
    (off by at most 2.1 * 2^-11 each, with what x A^T adds), so a score is off by
    d <= 4.4 * 2^-11 sum |q k|; softmax weights by a factor within e^(+-2d); P,
    v (once, with x A^T) and the output are rounded to f16: together
    (2d + d^2 + 3.2 * 2^-11) max |v|."""
    layer, lens, who = 1, [100, 64, 128, 30], [0, 2, -1, 1]
    R = sum(lens)
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(R, 1024, generator=g, device="cuda").half()
    w = torch.from_numpy(weight(header, arch.wqkv(layer))).cuda().half()
    lora = ops.Lora(ops.F16, 1024, 3072, w.data_ptr(), 1024, slots=3, max_rank=48)
    mats = {}
    for s in RANKS:
        a, b = matrices(s, arch.wqkv(layer))
        lora.set(s, a, b, SCALE[s])
        mats[s] = [torch.from_numpy(v).cuda().double() for v in (a, b)]
    sc = ops.RopeScaling(ops.ROPE_LINEAR, 2.0)
    freqs, m = ops.rope_freqs(modelgen.THETA_SLIDING, 64, sc)
    qkv = torch.empty(R, 3072, device="cuda", dtype=torch.float16)
    pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).cuda()
    st = torch.cuda.current_stream().cuda_stream
    lora.run(lora.plan(lens, who), x.data_ptr(), 1024, qkv.data_ptr(), 3072, stream=st)
    spec = ops.RopeSpec(ops.F16, 64, 64, freqs, mscale=m * arch.SCALE)
    ops.rope(spec, [ops.RopeTensor(qkv.data_ptr(), qkv.data_ptr(), 32, 3072, 64, 3072, 64)], R, pos=pos.data_ptr(), stream=st)
    torch.cuda.synchronize()
    got = torch.from_numpy(E.selftest_attention(qkv.cpu().numpy(), lens, arch.WINDOW))
    y = x.double() @ w.double().T
    row = 0
    for n, s in zip(lens, who):
        if s >= 0:
            a, b = mats[s]
            y[row:row + n] += SCALE[s] * (x[row:row + n].double() @ a.T) @ b.T
        row += n
    ang = pos.double()[:, None] * torch.from_numpy(freqs).cuda()[None]
    c, s_ = ang.cos()[:, None], ang.sin()[:, None]
    y = y.view(R, 3, 16, 64)
    # both q and k carry the factor
    rot = lambda t: torch.cat([t[..., :32] * c - t[..., 32:] * s_, t[..., 32:] * c + t[..., :32] * s_], -1) * (m * arch.SCALE)
    q, k, v = rot(y[:, 0]), rot(y[:, 1]), y[:, 2]
    row = 0
    for n in lens:
        sl = slice(row, row + n)
        row += n
        sc_ = torch.einsum("qhd,khd->hqk", q[sl], k[sl])
        i = torch.arange(n, device="cuda")
        far = (i[:, None] - i[None]).abs() > arch.WINDOW
        want = torch.einsum("hqk,khd->qhd", sc_.masked_fill(far, float("-inf")).softmax(-1), v[sl]).reshape(n, 1024)
        mags = torch.einsum("qhd,khd->hqk", q[sl].abs(), k[sl].abs()).masked_fill(far, 0.0)
        d = 4.4 * 2.0 ** -11 * mags.amax(-1).T[..., None]                                 # [q, h, 1]
        tol = (2 * d + d * d + 3.2 * 2.0 ** -11) * v[sl].abs().amax(0)[None]              # [q, h, 64]
        err = (got[sl].cuda().double() - want).abs().view(n, 16, 64)
        assert bool((err <= tol).all()), float((err / tol).max())
