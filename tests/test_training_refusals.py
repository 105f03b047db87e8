"""Calls of trained attention, of the f32 attention's backward pass and of log-probabilities that are refused before anything is launched: the
library's host code on a runtime that runs nothing, so that no GPU is needed."""
import pytest

from test_kv_cache_refusals import answers, run, stub  # noqa: F401 (stub is a fixture)

SHAPE = "hip.AttentionTraining(2, 4, 100, 64, 0.125, kv_heads=2)"
FORWARD = f"shape={SHAPE}, q=1*M, ld_q=256, k=2*M, v=3*M, ld_kv=128, out=4*M, ld_out=256, lse=5*M"
BACKWARD = FORWARD + (", grad_out=6*M, ld_grad_out=256, grad_q=7*M, ld_grad_q=256, grad_k=8*M, grad_v=9*M, ld_grad_kv=128, grad_table=None")


def shape(text):
    return f"shape=hip.AttentionTraining({text})"


def biased(text):
    return shape(f"2, 4, 100, 64, 0.125, position_bias=hip.PositionBias({text}), kv_heads=2")


SHAPES = {
    shape("2, 4, 100, 64, 0.125, kv_heads=3"): "invalid", shape("2, 4, 100, 64, 0.125, kv_heads=0"): "invalid",
    shape("2, 4, 100, 32, 0.125, kv_heads=2"): "unsupported", shape("2, 4, 100, 96, 0.125, kv_heads=2"): "unsupported",
    shape("2, 4, 100, 256, 0.125, kv_heads=2"): "unsupported", shape("2, 4, 100, 64, float('nan'), kv_heads=2"): "nonfinite",
    shape("2, 4, 100, 64, float('inf'), kv_heads=2"): "nonfinite", shape("2, 4, 100, 64, 3e38, kv_heads=2"): "unsupported",
    shape("2, 4, 100, 64, -0.5, kv_heads=2"): "taken", shape("2, 4, 100, 64, 0.0, kv_heads=2, lengths=10*M"): "taken",
    shape("0, 4, 100, 64, 0.125, kv_heads=2"): "taken", shape("2, 0, 100, 64, 0.125, kv_heads=0"): "taken", shape("2, 4, 0, 64, 0.125, kv_heads=2"): "taken",
    shape("2**62, 4, 100, 64, 0.125, kv_heads=2"): "invalid", shape("2**31, 4, 1, 64, 0.125, kv_heads=2"): "unsupported",
    shape("1, 4, 2**31 - 300, 64, 0.125, kv_heads=2"): "unsupported", shape("1, 4, 2**22, 64, 0.125, kv_heads=2"): "unsupported",  # a sequence of 2 GiB
    biased("2, 100, 10*M"): "taken", biased("1, 100, 10*M"): "invalid", biased("2, 100, 10*M, bidirectional=True"): "invalid",
    biased("4, 2, 10*M, bidirectional=True"): "taken", biased("4, 2, 10*M"): "invalid", biased("5, 100, 10*M, bidirectional=True"): "invalid",
    biased("32, 8, 10*M, bidirectional=True"): "invalid", biased("32, 9, 10*M, bidirectional=True"): "taken", biased("256, 2048, 10*M"): "taken",
    biased("258, 2048, 10*M"): "unsupported", biased("256, 2049, 10*M"): "unsupported", biased("0, 100, 10*M"): "invalid", biased("8, 100, None"): "invalid",
}
ROWS = {
    "q=None": "invalid", "k=None": "invalid", "v=None": "invalid", "out=None": "invalid", "lse=None": "invalid", "ld_q=248": "invalid", "ld_kv=120": "invalid",
    "ld_out=192": "invalid", "ld_q=260": "unsupported", "ld_kv=132": "unsupported", "ld_out=257": "unsupported", "q=1*M + 8": "unsupported",
    "k=2*M + 2": "unsupported", "v=3*M + 4": "unsupported", "out=4*M + 8": "unsupported", "ld_q=2**31": "unsupported",
}


def test_forward(stub):  # noqa: F811
    expected = {"": "taken", **SHAPES, **ROWS, "out=1*M": "invalid", "out=2*M + 16": "invalid", "lse=3*M": "invalid", "lse=4*M": "invalid",
                # columns of one matrix of 512: queries, keys, values; the result beside them or not
                "q=1*M, k=1*M + 512, v=1*M + 768, ld_q=512, ld_kv=512": "taken", "ld_q=512, ld_out=512, out=1*M + 512": "taken",
                "ld_q=512, ld_out=512, out=1*M + 496": "invalid", "ld_q=512, ld_out=512, out=1*M + 528": "invalid",
                "ld_kv=512, ld_out=512, out=2*M + 256": "taken", "ld_kv=512, ld_out=512, out=2*M + 240": "invalid",
                f"{shape('2, 4, 100, 64, 0.125, kv_heads=2, lengths=4*M + 64')}": "invalid", biased("8, 100, 4*M + 64"): "invalid",
                biased("8, 100, 5*M + 3196"): "invalid", biased("8, 100, 5*M + 3200"): "taken"}
    assert answers(stub, "hip.attention_training_bf16_dev", FORWARD, expected) == list(expected.values())


def test_backward(stub):  # noqa: F811
    expected = {"": "taken", **SHAPES, **ROWS, "grad_out=None": "invalid", "grad_q=None": "invalid", "grad_k=None": "invalid", "grad_v=None": "invalid",
                "ld_grad_out=255": "invalid", "ld_grad_q=255": "invalid", "ld_grad_kv=127": "invalid", "ld_grad_q=257": "unsupported",
                "grad_out=6*M + 8": "unsupported", "grad_k=8*M + 8": "unsupported", "grad_table=11*M": "invalid",  # without a bias
                "grad_q=1*M": "invalid", "grad_q=6*M": "invalid", "grad_k=2*M": "invalid", "grad_v=3*M": "invalid", "grad_k=9*M": "invalid",
                "grad_v=5*M": "invalid", "out=6*M": "taken",  # both are read
                "grad_q=7*M, grad_k=7*M + 512, grad_v=7*M + 768, ld_grad_q=512, ld_grad_kv=512": "taken",
                "grad_q=7*M, grad_k=7*M + 512, grad_v=7*M + 752, ld_grad_q=512, ld_grad_kv=512": "invalid"}
    assert answers(stub, "hip.attention_backward_bf16_dev", BACKWARD, expected) == list(expected.values())
    expected = {"": "taken", "grad_table=None": "taken", "grad_table=10*M": "invalid", "grad_table=7*M": "invalid", "grad_table=10*M + 124": "invalid",
                "grad_table=10*M + 128": "taken", shape("2, 4, 0, 64, 0.125, kv_heads=2, position_bias=hip.PositionBias(8, 100, 10*M)"): "taken",
                shape("0, 4, 9, 64, 0.125, kv_heads=2, position_bias=hip.PositionBias(8, 100, None)"): "taken"}
    base = BACKWARD.replace(SHAPE, biased("8, 100, 10*M")[6:]).replace("grad_table=None", "grad_table=11*M")
    assert answers(stub, "hip.attention_backward_bf16_dev", base, expected) == list(expected.values())


def test_empty_shapes_launch_nothing_but_a_table_of_zeros(stub):  # noqa: F811
    assert run(stub, f"""
for text, table in (("hip.AttentionTraining(0, 4, 9, 64, 1.0)", None), ("hip.AttentionTraining(2, 4, 0, 64, 1.0)", None),
                    ("hip.AttentionTraining(0, 4, 9, 64, 1.0, position_bias=hip.PositionBias(8, 100, 10*M))", 11*M)):
    before = launches.value
    hip.attention_training_bf16_dev(eval(text), None, 0, None, None, 0, None, 0, None)
    hip.attention_backward_bf16_dev(eval(text), None, 0, None, None, 0, None, 0, None, None, 0, None, 0, None, None, 0, table)
    print(launches.value - before)
""") == ["0", "0", "1"]


def test_scratch_that_cannot_be_had(stub):  # noqa: F811
    """The backward passes and cut rows need scratch memory: a runtime error, and nothing launched."""
    assert run(stub, f"""
def status(call, *args):
    before = launches.value
    try:
        call(*args)
    except hip.HipErr as e:
        return (e.status, launches.value - before)
    return "taken"
hip.init()
no_memory.value = 1
print(status(hip.attention_backward_bf16_dev, {SHAPE}, 1*M, 256, 2*M, 3*M, 128, 4*M, 256, 5*M, 6*M, 256, 7*M, 256, 8*M, 9*M, 128),
      status(hip.attention_backward_f32_dev, 2, 100, 64, 0.1, False, 1*M, 2*M, 3*M, None, None, 4*M, 5*M, 6*M, 7*M, 8*M),
      status(hip.token_log_probs_f32_dev, 1, 100000, 1*M, 100000, 2*M, 3*M, 4*M, 5*M), sep=";")
""") == ["(3,", "0);(3,", "0);(3,", "0)"]


def test_f32_backward(stub):  # noqa: F811
    base = ("contexts=2, sequence=50, head_dim=64, scale=0.125, causal=True, q=1*M, k=2*M, v=3*M, z_bias=4*M, attn_bias=5*M, out=6*M, grad_out=7*M, "
            "grad_q=8*M, grad_k=9*M, grad_v=10*M, grad_z_bias=11*M, grad_attn_bias=12*M")
    expected = {"": "taken", "causal=False": "taken", "grad_z_bias=None": "taken", "grad_attn_bias=None": "taken", "z_bias=None": "invalid",
                "attn_bias=None": "invalid", "z_bias=None, grad_z_bias=None, attn_bias=None, grad_attn_bias=None": "taken",
                **{f"{name}=None": "invalid" for name in ("q", "k", "v", "out", "grad_out", "grad_q", "grad_k", "grad_v")},
                "scale=float('nan')": "nonfinite", "scale=0.0": "taken", "head_dim=257": "unsupported", "head_dim=256": "taken", "head_dim=1": "taken",
                "contexts=0, q=None": "taken", "sequence=0, q=None": "taken", "contexts=2**31, sequence=1": "unsupported", "sequence=2**31": "unsupported",
                "sequence=2**23, z_bias=None, grad_z_bias=None, attn_bias=None, grad_attn_bias=None, contexts=1": "unsupported", "contexts=2**62": "invalid",
                "sequence=2**32, contexts=2**31": "invalid", "grad_q=1*M": "invalid", "grad_k=2*M + 25596": "invalid", "grad_k=2*M + 25600": "taken",
                "grad_v=8*M": "invalid", "grad_z_bias=4*M + 396": "invalid", "grad_attn_bias=5*M": "invalid", "grad_z_bias=12*M + 16": "invalid", "q=2*M": "taken",
                "head_dim=0, q=None, k=None, v=None, out=None, grad_out=None, grad_q=None, grad_k=None, grad_v=None": "taken"}
    assert answers(stub, "hip.attention_backward_f32_dev", base, expected) == list(expected.values())


@pytest.mark.parametrize("kind,size", [("f32", 4), ("bf16", 2)])
def test_log_probs(stub, kind, size):  # noqa: F811
    base = ("rows=10, vocab=100, logits=1*M, ld=100, tokens=2*M, log_probs=3*M, entropies=4*M, normalizers=5*M, top=5, top_ids=6*M, top_log_probs=7*M")
    expected = {"": "taken", "rows=0, logits=None": "taken", "vocab=0": "invalid", "ld=99": "invalid", "ld=101": "taken", "logits=None": "invalid",
                "tokens=None": "invalid", "tokens=None, log_probs=None": "taken", "entropies=None": "taken", "normalizers=None": "taken", "top_ids=None": "invalid",
                "top_log_probs=None": "invalid", "top=0, top_ids=None, top_log_probs=None": "taken", "top=101": "invalid", "top=33": "unsupported", "top=32": "taken",
                "vocab=3, top=4": "invalid", "rows=2**31": "unsupported", "vocab=2**31, ld=2**31": "unsupported", "rows=2**31 - 1, ld=2**62": "invalid",
                "logits=1*M + 1": "invalid", f"logits=1*M + {size}": "taken", f"log_probs=1*M + {1000 * size - 2}": "invalid",
                f"log_probs=1*M + {1000 * size}": "taken", "entropies=2*M + 36": "invalid", "entropies=3*M": "invalid", "top_ids=7*M + 196": "invalid",
                "tokens=None, log_probs=None, entropies=None, normalizers=None, top=0, top_ids=None, top_log_probs=None": "taken"}
    assert answers(stub, f"hip.token_log_probs_{kind}_dev", base, expected) == list(expected.values())
    base = ("rows=10, vocab=100, logits=1*M, ld=100, tokens=2*M, normalizers=3*M, entropies=4*M, grad_log_probs=5*M, grad_entropies=6*M, grad_logits=7*M, "
            "ld_grad=100")
    expected = {"": "taken", "rows=0, grad_logits=None": "taken", "vocab=0": "invalid", "logits=None": "invalid", "grad_logits=None": "invalid",
                "normalizers=None": "invalid", "tokens=None": "invalid", "tokens=None, grad_log_probs=None": "taken", "entropies=None": "invalid",
                "entropies=None, grad_entropies=None": "taken", "ld_grad=99": "invalid", "grad_logits=1*M": "taken", "grad_logits=1*M, ld_grad=104": "invalid",
                "grad_logits=1*M, ld_grad=104, rows=1": "taken", f"grad_logits=1*M + {size}": "invalid", "grad_logits=3*M": "invalid", "grad_logits=2*M + 8": "invalid",
                f"ld=208, ld_grad=208, grad_logits=1*M + {100 * size}": "taken", f"ld=208, ld_grad=208, grad_logits=1*M + {99 * size}": "invalid",
                "rows=2**31": "unsupported", "grad_logits=7*M + 1": "invalid"}
    assert answers(stub, f"hip.token_log_probs_backward_{kind}_dev", base, expected) == list(expected.values())


def test_more_workgroups_than_a_launch_has(stub):  # noqa: F811
    """A launch counts its threads in 32 bits: 2^24 workgroups of 256 are one too many."""
    far = "logits=M, ld=1, tokens=2**40, log_probs=2**41, entropies=None, normalizers=None, top=0, top_ids=None, top_log_probs=None"
    assert answers(stub, "hip.token_log_probs_f32_dev", f"rows=2**24 - 1, vocab=1, {far}", {"": "taken", "rows=2**24": "unsupported"}) == ["taken", "unsupported"]
    back = "logits=M, ld=1, tokens=None, normalizers=2**40, entropies=None, grad_log_probs=None, grad_entropies=None, grad_logits=2**41, ld_grad=1"
    expected = {"": "taken", "rows=2**24": "unsupported"}
    assert answers(stub, "hip.token_log_probs_backward_bf16_dev", f"rows=2**24 - 1, vocab=1, {back}", expected) == list(expected.values())
    wide = "q=M, ld_q=64, k=2**41, v=2**42, ld_kv=64, out=2**43, ld_out=64, lse=2**44"
    expected = {"": "taken", shape("2**24, 1, 1, 64, 0.125"): "unsupported", shape("2**23, 1, 129, 64, 0.125"): "unsupported",
                shape("2**23 - 1, 2, 1, 64, 0.125, kv_heads=1") + ", ld_q=128, ld_out=128": "taken",
                shape("1, 2**14, 1, 64, 0.125, position_bias=hip.PositionBias(8, 100, 2**45)") + ", ld_q=2**20, ld_kv=2**20, ld_out=2**20": "unsupported"}
    assert answers(stub, "hip.attention_training_bf16_dev", f"{shape('2**24 - 1, 1, 1, 64, 0.125')}, {wide}", expected) == list(expected.values())
    base = ("contexts=2**24 - 1, sequence=1, head_dim=1, scale=1.0, causal=False, q=M, k=2**41, v=2**42, z_bias=None, attn_bias=None, out=2**43, grad_out=2**44, "
            "grad_q=2**45, grad_k=2**46, grad_v=2**47")
    expected = {"": "taken", "contexts=2**24": "unsupported", "contexts=2**23, sequence=33": "unsupported"}
    assert answers(stub, "hip.attention_backward_f32_dev", base, expected) == list(expected.values())
