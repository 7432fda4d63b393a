"""The 4-bit engine in the harness that measures: steps, and a profile with the rates of all kernels that the 4 bits bring."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weight_bits,kv_bits", [(4, 4), (16, 4), (4, 16)])
def test_steps_and_profiles_of_a_4_bit_engine(weight_bits, kv_bits):
    from carbon_engine_b200.bench_support import BenchHarness
    cfg = dict(num_hidden_layers=2, hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64, intermediate_size=512, vocab_size=512,
               max_position_embeddings=4096, rms_norm_eps=1e-6, rope_theta=10000.0, tie_word_embeddings=False, torch_dtype="bfloat16")
    h = BenchHarness(cfg, max_batch=3, context=100, new_tokens=64, step_tokens=256, weight_bits=weight_bits, kv_bits=kv_bits)
    assert h.decode(3, 4, 3)["tokens_per_s"] > 0
    got = h.profile(3, 200, 1e4, 1e4)
    for part in ("decode", "prefill"):
        rows = {r["kernel"].split(" ")[0]: r for r in got[part]["kernels"]}
        rated = [n for n in rows if n.startswith("int4_")]
        assert rated and all(rows[n]["gb_s"] > 0 for n in rated), rows
        assert ("int4_kv_write_kernel" in rows) == (kv_bits == 4) and any("int4_attention" in n for n in rows) == (kv_bits == 4)
        weights = {"decode": "int4_stream_kernel", "prefill": "int4_dequantise_weight_kernel"}[part]
        assert (weights in rows) == (weight_bits == 4)


def test_work_of_attention_with_a_window():
    from types import SimpleNamespace
    from carbon_engine_b200 import ops_int4
    from carbon_engine_b200.parts.attention import PagedAttention
    m = PagedAttention(hidden=256, heads=4, kv_heads=2, head_dim=64, window=10, prefix="a")
    ctx = SimpleNamespace(h_q_start=[0, 1, 4], h_ctx_before=[20, 5])
    pages = ops_int4.Int4Pages(1, 2, 16, 64, 32)
    # one token of 10 keys; three, of 6, 7 and 8 keys, 8 in all
    assert m.int4_work(ctx, pages, 2, 0, 1) == (10 * pages.bytes_per_token() + 2 * 256 * 2, 4 * 10 * 256)
    assert m.int4_work(ctx, pages, 2, 1, 2) == (8 * pages.bytes_per_token() + 2 * 3 * 256 * 2, 4 * 21 * 256)
