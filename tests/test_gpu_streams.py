"""A context on the caller's stream: its ops take their turn among torch's, with no
synchronisation on either side.
"""
import numpy as np
import pytest

import intllm
import serve_plain as P
import spec

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def streams():
    return [torch.cuda.default_stream(0), torch.cuda.Stream(0)]


def rows(rng, T, V):
    return (rng.standard_normal((T, V)) * (2.5 * P.ONE)).astype(np.int64)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("T,V", [(40, 2000), (2, 12000)])
def test_calls_between_torch_operations(which, T, V):
    """Inputs that torch is still making when the op is enqueued, results that torch reads
    and inputs that it overwrites right behind it."""
    rng = np.random.default_rng(V)
    x = rows(rng, T, V)
    tokens = rng.integers(0, V, T).astype(np.int32)
    host = torch.from_numpy(x).pin_memory()
    s = streams()[which]
    with torch.cuda.stream(s), intllm.Context(0, stream=s.cuda_stream) as c:
        big = torch.randn(8192, 8192, device=DEV)
        tok = torch.from_numpy(tokens).to(DEV)
        first = torch.zeros(T, V, dtype=torch.int64, device=DEV)
        ent = torch.zeros(T, dtype=torch.int64, device=DEV)
        c.logprobs_rows(first.data_ptr(), T, V, None, None, ent.data_ptr())   # (its workspace)
        for _ in range(3):
            d = torch.zeros(T, V, dtype=torch.int64, device=DEV)
            logp, ent = torch.zeros(2, T, dtype=torch.int64, device=DEV)
            for _ in range(4):                 # tens of milliseconds of torch's own work
                big = torch.mm(big, big) * 1e-4
            d.copy_(host, non_blocking=True)
            c.logprobs_rows(d.data_ptr(), T, V, tok.data_ptr(), logp.data_ptr(), ent.data_ptr())
            got = torch.stack([logp, ent]) + 1
            d.zero_()
            want = P.logprobs(x, tokens, 0)
            assert (got[0].cpu().numpy() == want[0] + 1).all()
            assert (got[1].cpu().numpy() == want[1] + 1).all()


@pytest.mark.parametrize("which", [0, 1])
def test_store_attend_and_read_back(which):
    """A cache in torch's memory, written and attended to on torch's stream."""
    rng = np.random.default_rng(which)
    nh, nkv, hd, T, p0 = 8, 2, 64, 9, 1200
    K, V = (rng.standard_normal((2, p0 + T, nkv, hd)) * P.ONE).astype(np.int64)
    qkv = (rng.standard_normal((T, nh + 2 * nkv, hd)) * P.ONE).astype(np.int64)
    s = streams()[which]
    with torch.cuda.stream(s), intllm.Context(0, stream=s.cuda_stream) as c:
        codes, steps = intllm.qcache_bytes(8, 1, p0 + T, nkv, hd)
        k, v = torch.zeros(2, codes, dtype=torch.uint8, device=DEV)
        ks, vs = torch.zeros(2, steps // 8, dtype=torch.int64, device=DEV)
        cache = c.qcache(*(t.data_ptr() for t in (k, v, ks, vs)), 8, 1, p0 + T, nkv, hd)
        dk, dv, x = (torch.from_numpy(a).pin_memory().to(DEV, non_blocking=True)
                     for a in (K, V, qkv))
        out = torch.zeros(T, nh, hd, dtype=torch.int64, device=DEV)
        c.qcache_store_rows(cache, 0, 0, p0 + T, dk.data_ptr(), dv.data_ptr(), nkv * hd)
        c.attn_rows_qcache(out.data_ptr(), x.data_ptr(), cache, 0, p0, T, nh)
        got = out.cpu().numpy()
        kv, vv = (P.values(*P.quantise(a, 8)) for a in (K, V))
        see = np.concatenate([np.ones((T, p0), bool), np.tri(T, dtype=bool)], 1)
        assert (got == P.attend(qkv[:, :nh], kv, vv, see)).all()
        codes = P.pack(P.quantise(K, 8)[0], 8)
        assert (k.cpu().numpy().reshape(codes.shape) == codes).all()


def test_graphs_on_a_lent_stream():
    """The context's own capture on the caller's stream, replayed between torch's work; the
    default stream has none."""
    rng = np.random.default_rng(4)
    lib = intllm.hip_lib()
    T, V = 3, 12000
    s = streams()[1]
    with torch.cuda.stream(s), intllm.Context(0, stream=s.cuda_stream) as c:
        d = torch.zeros(T, V, dtype=torch.int64, device=DEV)
        ent = torch.zeros(T, dtype=torch.int64, device=DEV)

        def call():
            c.logprobs_rows(d.data_ptr(), T, V, None, None, ent.data_ptr())

        call()
        intllm.check("begin", lib.q48_graph_begin(c.h))
        call()
        intllm.check("end", lib.q48_graph_end(c.h))
        for _ in range(3):
            x = rows(rng, T, V)
            d.copy_(torch.from_numpy(x).pin_memory(), non_blocking=True)
            intllm.check("launch", lib.q48_graph_launch(c.h, 1))
            got = ent.cpu().numpy()
            call()
            assert (ent.cpu().numpy() == got).all()
            assert (got == P.logprobs(x, np.zeros(T, np.int64), 0)[1]).all()
        intllm.check("drop", lib.q48_graph_drop(c.h))
    with intllm.Context(0, stream=0) as c:
        assert lib.q48_graph_begin(c.h) == intllm.Q48_ESTATE
        assert lib.q48_graph_capture(c.h) == intllm.Q48_ESTATE
        b = c.to_device(np.arange(6))          # and no error is left behind
        c.add(b.ptr, b.ptr, 6)
        assert (b.download() == 2 * np.arange(6)).all()


def test_the_caller_s_capture_takes_what_needs_no_workspace():
    rng = np.random.default_rng(5)
    lib = intllm.hip_lib()
    T, V, W = 3, 500, 12000
    s = streams()[1]
    with torch.cuda.stream(s), intllm.Context(0, stream=s.cuda_stream) as c:
        c.rope_init(64, 400, 10000)
        d = torch.zeros(T, V, dtype=torch.int64, device=DEV)
        wide = torch.zeros(1, W, dtype=torch.int64, device=DEV)
        ent = torch.zeros(T, dtype=torch.int64, device=DEV)
        kv = torch.zeros(2, 400, 2, 64, dtype=torch.int64, device=DEV)
        q, o, n = torch.zeros(3, 8, 64, dtype=torch.int64, device=DEV)
        c.logprobs_rows(wide.data_ptr(), 1, W, None, None, ent.data_ptr())   # (its workspace)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            c.logprobs_rows(d.data_ptr(), T, V, None, None, ent.data_ptr())
            refused = [lib.q48_logprobs_rows(c.h, wide.data_ptr(), 1, W, None, None,
                                             ent.data_ptr(), 0, None, None),
                       lib.q48_attn_decode_rope(c.h, o.data_ptr(), q.data_ptr(), kv[0].data_ptr(),
                                                kv[1].data_ptr(), n.data_ptr(), n.data_ptr(), 0,
                                                390, 8, 2, 64, 400),
                       lib.q48_graph_capture(c.h)]
            try:
                intllm.Context(0, stream=s.cuda_stream)
            except intllm.Q48Error as e:
                refused.append(e.code)
        assert refused == [intllm.Q48_ESTATE] * 4, refused
        for _ in range(3):
            x = rows(rng, T, V)
            d.copy_(torch.from_numpy(x))
            ent.zero_()
            graph.replay()
            assert (ent.cpu().numpy() == P.logprobs(x, np.zeros(T, np.int64), 0)[1]).all()


def test_the_host_s_decode_on_a_lent_stream():
    """Generation through the C host: the same tokens and hashes on the context's own
    stream, on the caller's, and on the default one, which has no graphs."""
    cfg = intllm.Config(*spec.TINY)
    prompt = spec.prompt(spec.SEED_TINY, 16, spec.TINY[6])
    ran = []
    for stream in (None, torch.cuda.Stream(0).cuda_stream, 0):
        with intllm.Context(0, stream=stream) as c:
            m = intllm.HostModel(c, cfg)
            m.synth(spec.SEED_TINY, 8)
            if stream == 0:
                with pytest.raises(intllm.Q48Error) as e:
                    m.decode_graph_hashed(5, 0, 8)
                assert e.value.code == intllm.Q48_ESTATE
                m.kv_reset()
            toks, hs, _ = m.generate(prompt, 8)
            graph = None
            if stream != 0:
                m.kv_reset()
                graph = m.decode_graph_hashed(5, 0, 8)[:3]
            ran.append((toks, hs, graph))
            m.free()
    assert ran[0] == ran[1] and ran[0][:2] == ran[2][:2]
