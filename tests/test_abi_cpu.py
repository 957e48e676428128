"""CPU-side checks of the product libraries (no GPU needed).

- libintllm_hip.so loads and exports every entry point include/intllm_hip.h
  declares; libq48host.so every q48h_* of host/q48_host.h.
- Argument validation happens before any device work (NULL context etc.).
- The host's config.json parsing matches load_config_json
  (llama_int.c:819-903): keys, defaults, null, float-like values, checks.
- The .mgw writer produces mgw_export's layout (llama_int.c:385-454,
  1718-1904), and — where the reference harness is built — the
  reference's own mgw_load accepts it and computes the same logits.
"""
import ctypes as C
import os
import re
import struct
import tempfile
from pathlib import Path

import numpy as np
import pytest

import intllm
import oracle_lib as O
import spec

ROOT = Path(__file__).resolve().parents[1]


def declared(header: Path, prefix: str):
    text = re.sub(r"/\*.*?\*/", "", header.read_text(), flags=re.S)
    return sorted(set(re.findall(r"\b(" + prefix + r"\w+)\s*\(", text)))


def test_hip_lib_exports_every_declared_symbol():
    lib = intllm.hip_lib()
    names = declared(ROOT / "include" / "intllm_hip.h", "q48_")
    assert len(names) >= 20
    for n in names:
        assert hasattr(lib, n), n


def test_host_lib_exports_every_declared_symbol():
    lib = intllm.host_lib()
    names = declared(ROOT / "int-llm_amd" / "host" / "q48_host.h", "q48h_")
    assert len(names) >= 15
    for n in names:
        assert hasattr(lib, n), n


def test_null_context_is_rejected_without_device_work():
    lib = intllm.hip_lib()
    assert lib.q48_gemv(None, None, None, None, 1, 1) == intllm.Q48_EINVAL
    assert lib.q48_rmsnorm(None, None, None, None, 4) == intllm.Q48_EINVAL
    assert lib.q48_sync(None) == intllm.Q48_EINVAL
    assert lib.q48_ctx_create(None, 0) == intllm.Q48_EINVAL
    assert intllm.strerror(intllm.Q48_ERANGE) == "token or position out of range"


def parse(text):
    c = intllm.Config()
    rc = intllm.host_lib().q48h_config_from_json_text(text.encode(), C.byref(c))
    return rc, c


def test_config_json_parsing_matches_load_config_json():
    rc, c = parse('{"architectures": ["LlamaForCausalLM"], "hidden_size": 2048, '
                  '"num_attention_heads": 32, "num_key_value_heads": 4, "num_hidden_layers": 22, '
                  '"intermediate_size": 5632, "vocab_size": 32000, '
                  '"max_position_embeddings": 2048, "rope_theta": 10000.0}')
    assert rc == 0 and c.as_tuple() == spec.TINYLLAMA
    # defaults: kv heads = heads, max_pos 2048, theta 10000; null -> default
    rc, c = parse('{"hidden_size": 256, "num_attention_heads": 8, "num_hidden_layers": 2,'
                  '"intermediate_size": 688, "vocab_size": 512, "rope_theta": null}')
    assert rc == 0 and (c.n_kv_heads, c.max_seq, c.rope_theta, c.head_dim) == (8, 2048, 10000, 32)
    # missing required field, indivisible heads, bad GQA ratio
    assert parse('{"hidden_size": 256}')[0] == -2
    assert parse('{"hidden_size": 250, "num_attention_heads": 8, "num_hidden_layers": 2,'
                 '"intermediate_size": 688, "vocab_size": 512}')[0] == -2
    assert parse('{"hidden_size": 256, "num_attention_heads": 8, "num_key_value_heads": 3,'
                 '"num_hidden_layers": 2, "intermediate_size": 688, "vocab_size": 512}')[0] == -2
    with tempfile.TemporaryDirectory() as d:
        assert intllm.host_lib().q48h_config_from_json(d.encode(), C.byref(intllm.Config())) == -1


def test_mgw_layout():
    cfg = intllm.Config(*spec.TINY)
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, "t.mgw")
        assert intllm.host_lib().q48h_mgw_write_synth(path.encode(), C.byref(cfg), 7, 4) == 0
        data = Path(path).read_bytes()
    magic, ver, endian, nt, ioff, doff = struct.unpack_from("<4sIIIQQ", data, 0)
    assert (magic, ver, endian, ioff) == (b"MGW\0", 1, 0x01020304, 128)
    assert nt == 3 + 9 * cfg.n_layers and doff == (128 + 96 * nt + 7) // 8 * 8
    cv = struct.unpack_from("<10i", data, 64)
    assert cv[:9] == spec.TINY and cv[9] == 0
    names, cur = [], doff
    for i in range(nt):
        e = data[ioff + 96 * i: ioff + 96 * (i + 1)]
        name = e[:64].split(b"\0")[0].decode()
        ne, off, nd = struct.unpack_from("<QQI", e, 64)
        assert off == cur and off % 8 == 0
        cur += 8 * ne
        names.append(name)
        # the data is the synthetic tensor of that name
        if name in ("model.norm.weight", "model.layers.1.self_attn.k_proj.weight"):
            rows = 1 if nd == 1 else struct.unpack_from("<I", e, 84)[0]
            got = np.frombuffer(data, dtype=np.int64, count=ne, offset=off)
            assert np.array_equal(got, O.synth(name, rows, ne // rows, 7, spec.SIGMA_W, 1))
    assert cur == len(data)
    assert names[:3] == ["model.embed_tokens.weight", "model.norm.weight", "lm_head.weight"]
    assert names[3] == "model.layers.0.input_layernorm.weight"


@pytest.mark.skipif(not O.REF_SO.exists(), reason="reference harness not built (needs /root/reference)")
def test_reference_mgw_load_accepts_written_file():
    """The reference's mgw_load reads the host-written file and its
    llama_forward gives the logits of the synthetic model."""
    lib = C.CDLL(str(O.REF_SO))
    lib.q48r_model_load_mgw.restype = C.c_void_p
    lib.q48r_model_load_mgw.argtypes = [C.c_char_p]
    lib.q48r_forward.argtypes = [C.c_void_p, C.c_int, C.c_int, C.c_void_p]
    lib.q48r_model_free_mgw.argtypes = [C.c_void_p]
    cfg = intllm.Config(*spec.TINY)
    om = O.Model(spec.TINY, 11)
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, "t.mgw")
        assert intllm.host_lib().q48h_mgw_write_synth(path.encode(), C.byref(cfg), 11, 4) == 0
        m = lib.q48r_model_load_mgw(path.encode())
        assert m
        for pos, tok in enumerate([5, 100, 511]):
            lg = np.empty(cfg.vocab, dtype=np.int64)
            assert lib.q48r_forward(m, tok, pos, lg.ctypes.data) == 0
            rc, want = om.forward(tok, pos)
            assert rc == 0 and np.array_equal(lg, want)
        lib.q48r_model_free_mgw(m)
    om.free()


def test_a_context_on_a_stream_is_refused_without_device_work():
    lib = intllm.hip_lib()
    assert lib.q48_ctx_create_on(None, 0, None) == intllm.Q48_EINVAL
    h = C.c_void_p(5)
    assert lib.q48_ctx_create_on(C.byref(h), -1, None) == intllm.Q48_EINVAL
    assert h.value is None
