"""4-bit serving ops and beam selection on streams of their own, in captured graphs, and over memory past 4 GiB. The same
kernels run in every setting, so their results must equal the plain eager call's bit for bit."""
import numpy as np
import pytest
import torch

from oracle import q4 as O

pytestmark = pytest.mark.gpu


def inputs(lk, seed, cap=4096):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = lk.Tensor
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    q4 = lk.ops.q4_gpu
    d = {"x": T(rand(3, 512).half()), "qkv": T(rand(3, (16 + 16) * 128).half()), "g": T((1 + 0.1 * rand(128)).half()),
         "q": T(rand(3, 16 * 128).half()), "w": q4.pack_w4(T((rand(512, 700) / 20).half())),
         "kv": q4.kv4_cache(3, 8, cap), "pos": T(torch.tensor([cap - 9, 70, 1000], device="cuda")),
         "logits": T(rand(3, 30000)), "scores": T(-torch.rand(3, device="cuda", generator=g)),
         "done": T(torch.tensor([0, 1, 0], device="cuda")), "n": T(torch.tensor([900], device="cuda"))}
    k, v = (T(rand(3 * (cap - 4), 8 * 128).half()) for _ in range(2))
    q4.kv4_write_f16_gpu(d["kv"], k, v, T(torch.zeros(3, dtype=torch.int64, device="cuda")))
    return d


def step(lk, d, kv):
    """One call of each op, over a given copy of the cache."""
    q4, T = lk.ops.q4_gpu, lk.Tensor
    y = q4.gemm_w4_f16_gpu(d["x"], d["w"])
    q = q4.qknorm_rope_kv4_f16_gpu(d["qkv"], d["g"], d["g"], d["pos"], kv)
    a = q4.attention_kv4_f16_gpu(q, kv, d["pos"])
    s, parent, tok, done = lk.ops.beam_select_f32_gpu(d["logits"], d["scores"], d["done"], 3, (7, 11))
    wide = q4.attention_kv4_f16_gpu(T(d["q"].t.repeat(20, 1)), kv, T(d["pos"].t.clamp(max=500)))  # rows of many workgroups
    q4.kv4_reorder_gpu(T(kv.t.unsqueeze(0)), parent, d["n"])
    return [x.t for x in (y, q, a, s, parent, tok, done, wide)] + [kv.t]


def eager(lk, d):
    out = [t.clone() for t in step(lk, d, lk.Tensor(d["kv"].t.clone()))]
    torch.cuda.synchronize()
    return out


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_streams_at_once(gpu):
    lk = gpu
    sets = [inputs(lk, 1), inputs(lk, 2)]
    want = [eager(lk, d) for d in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for d, s in zip(sets, streams):
            with torch.cuda.stream(s):
                got.append(step(lk, d, lk.Tensor(d["kv"].t.clone())))
        for s in streams:
            s.synchronize()
        for g, w in zip(got, want):
            assert same(g, w)


def test_graphs_replayed_on_two_streams(gpu):
    """Two captured graphs, replayed together and apart, with eager work between; new inputs written in place."""
    lk = gpu
    sets = [inputs(lk, 3), inputs(lk, 4)]
    want = [eager(lk, d) for d in sets]
    graphs, outs, caches = [], [], []
    for d in sets:
        kv = lk.Tensor(d["kv"].t.clone())
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            outs.append(step(lk, d, kv))
        graphs.append(graph)
        caches.append(kv)
    streams = [torch.cuda.Stream() for _ in sets]
    other = inputs(lk, 5)
    for rep in range(6):
        for d, kv in zip(sets, caches):
            kv.t.copy_(d["kv"].t)
        eager(lk, other)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams if rep % 2 else [torch.cuda.current_stream()] * 2):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert same(o, w), rep
    # other inputs through the first graph
    for name in ("x", "qkv", "q", "logits", "scores", "done", "n", "pos", "g"):
        sets[0][name].t.copy_(other[name].t)
    sets[0]["w"].q.t.copy_(other["w"].q.t)
    sets[0]["w"].s.t.copy_(other["w"].s.t)
    caches[0].t.copy_(other["kv"].t)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert same(outs[0], eager(lk, other))


def test_caches_past_4_gib(gpu):
    """One sequence of 8 heads and 4 Mi rows (4.8 GB): the last head's values lie past 4 GiB. Rows of zeros but three, so the
    softmax has a closed form."""
    lk, q4 = gpu, gpu.ops.q4_gpu
    cap, kvh = 1 << 22, 8
    kv = q4.kv4_cache(1, kvh, cap)
    assert kv.nbytes > 1 << 32
    r = np.random.default_rng(6)
    at = [5, 1 << 20, cap - 1]
    k, v = np.zeros((3, kvh * 128), np.float16), np.zeros((3, kvh * 128), np.float16)
    k[:] = 0.5 * r.integers(-1, 2, k.shape)
    v[:] = r.integers(-1, 2, v.shape)
    pos = lambda p: lk.Tensor(torch.tensor([p], device="cuda"))  # noqa: E731
    G = lambda a: lk.from_numpy(a, device="gpu", copy=True)  # noqa: E731
    for i, p in enumerate(at):
        q4.kv4_write_f16_gpu(kv, G(k[i:i + 1]), G(v[i:i + 1]), pos(p))
    held = O.cache_values(k, v, kvh)
    read = q4.kv4_read_f16_gpu(lk.Tensor(kv.t[0, 1, kvh - 1])).t[torch.tensor(at)].cpu().numpy()
    assert np.array_equal(read.astype(np.float64), held[1][:, kvh - 1])
    for t in (1, 40):
        q = np.tile((4 * k.astype(np.float32).reshape(3, kvh, 128).sum(0)).reshape(1, -1), (t, 1)).astype(np.float16)
        got = q4.attention_kv4_f16_gpu(G(q), kv, pos(cap - t)).t[-1].cpu().numpy().reshape(kvh, 128).astype(np.float64)
        for h in range(kvh):
            s = held[0][:, h] @ q[0].reshape(kvh, 128)[h].astype(np.float64) / np.sqrt(128)
            m = max(s.max(), 0)
            e = np.exp(s - m)
            ref = e @ held[1][:, h] / (e.sum() + (cap - 3) * np.exp(-m))
            # weights as in test_q4_gpu, and a sum of 4 Mi f32 terms over lanes, waves and key ranges
            assert np.abs(got[h] - ref).max() <= 2.0 ** -11 * np.abs(ref).max() + 2.0 ** -22 * (8 + np.sqrt(cap))


def test_reorder_past_4_gib(gpu):
    """Two layers of two sequences of 8 heads and 2 Mi rows (9.7 GB): the last head's values of the last sequence."""
    q4 = gpu.ops.q4_gpu
    cap = 1 << 21
    kv = q4.kv4_cache(2, 8, cap, layers=2)
    assert kv.nbytes > 1 << 33
    kv.t[:, 0].fill_(7)
    n = 45
    i64 = lambda *v: gpu.Tensor(torch.tensor(v, device="cuda"))  # noqa: E731
    q4.kv4_reorder_gpu(kv, i64(0, 0), i64(n))
    codes = kv.t[..., : 64 * cap].unflatten(-1, (cap, 64))
    scales = kv.t[..., 64 * cap:].unflatten(-1, (4, cap, 2))
    for part, rows in ((codes[:, 1], -2), (scales[:, 1], -2)):
        assert (part.narrow(rows, 0, n) == 7).all() and (part.narrow(rows, n, 200) == 0).all()


def test_weights_past_4_gib(gpu):
    """K = 4096, N = 2.2 million: 4.5 GB of codes; the last columns against the same columns as a weight of their own."""
    lk, q4 = gpu, gpu.ops.q4_gpu
    k, tiles = 4096, 137500
    q = torch.randint(-2 ** 31, 2 ** 31 - 1, (tiles, k // 128, 256), dtype=torch.int32, device="cuda")
    s = torch.full((tiles, k // 128, 16, 1), 2.0 ** -6, dtype=torch.float16, device="cuda")
    assert q.numel() * 4 > 1 << 32
    w = q4.PackedWeight4(lk.Tensor(q), lk.Tensor(s), (k, 16 * tiles), 128)
    end = q4.PackedWeight4(lk.Tensor(q[-40:]), lk.Tensor(s[-40:]), (k, 640), 128)
    v = q4.unpack_w4_f16_gpu(end).numpy().astype(np.float64)
    for m in (1, 20):
        x = np.random.default_rng(m).standard_normal((m, k)).astype(np.float16)
        got = q4.lm_head_w4_f16_gpu(lk.from_numpy(x, device="gpu", copy=True), w).t[:, -640:].cpu().numpy()
        x = x.astype(np.float64)
        ref, term = x @ v, 2.0 ** -22 * np.sqrt(k) * np.sqrt((x * x) @ (v * v))
        assert (np.abs(got - ref) <= 2.0 ** -23 * np.abs(ref) + term).all()
