"""What the operators at the two ends of the vocabulary refuse, before any launch: shapes, types and values by `ValueError`, CPU
tensors by the table's "strict_cuda" `RuntimeError`, and wrong arguments of the C ABI by its codes.  No GPU is needed."""
import ctypes as C

import pytest
import torch

from speedup_thingy_b200 import _abi as A
from speedup_thingy_b200 import kernels as K

X = torch.zeros(2, 3, 16)
TOK = torch.zeros(2, 3, dtype=torch.int64)
LIST = torch.zeros(2, 3, 4), torch.zeros(2, 3, 4, dtype=torch.int64)
W = torch.zeros(16, 8)


@pytest.mark.parametrize("call, message", [
    (lambda: K.k_token_logprobs(X.double(), TOK), "bf16, fp16 or fp32"),
    (lambda: K.k_token_logprobs(X.to(torch.int32), TOK), "bf16, fp16 or fp32"),
    (lambda: K.k_token_logprobs(torch.zeros(()), torch.zeros((), dtype=torch.int64)), "at least one column"),
    (lambda: K.k_token_logprobs(torch.zeros(2, 3, 0), TOK), "at least one column"),
    (lambda: K.k_token_logprobs(X, TOK[0]), "integer tokens"),
    (lambda: K.k_token_logprobs(X, TOK.float()), "integer tokens"),
    (lambda: K.k_token_logprobs(X, TOK, top_k=-1), "top_k must be in 0..16"),
    (lambda: K.k_token_logprobs(X, TOK, top_k=17), "top_k must be in 0..16"),
    (lambda: K.k_token_logprobs(torch.zeros(2, 3, 1000), TOK, top_k=257), "top_k must be in 0..256"),
    (lambda: K.k_token_logprobs(X, TOK, temperature=0.0), "temperature"),
    (lambda: K.k_token_logprobs(X, TOK, temperature=-1.0), "temperature"),
    (lambda: K.k_token_logprobs(X, TOK, temperature=float("nan")), "temperature"),
    (lambda: K.k_token_logprobs(X, TOK, temperature=float("inf")), "temperature"),
    (lambda: K.k_token_logprobs(X, TOK.to("meta")), "must be on cpu"),
    (lambda: K.k_distill_topk(X.double(), *LIST), "bf16, fp16 or fp32"),
    (lambda: K.k_distill_topk(X, LIST[0], LIST[1].float()), "integer ids"),
    (lambda: K.k_distill_topk(X, LIST[1], LIST[1]), "floating log probabilities"),
    (lambda: K.k_distill_topk(X, LIST[0][..., :3], LIST[1]), "ids [..., k]"),
    (lambda: K.k_distill_topk(X, LIST[0][0], LIST[1][0]), "ids [..., k]"),
    (lambda: K.k_distill_topk(X, LIST[0][..., :0], LIST[1][..., :0]), "lists of 1..256"),
    (lambda: K.k_distill_topk(X, torch.zeros(2, 3, 257), torch.zeros(2, 3, 257, dtype=torch.int64)), "lists of 1..256"),
    (lambda: K.k_distill_topk(X, *LIST, temperature=0.0), "temperature"),
    (lambda: K.k_distill_topk(X, LIST[0].to("meta"), LIST[1]), "must be on cpu"),
    (lambda: K.k_embedding(TOK, W.double()), "a table"),
    (lambda: K.k_embedding(TOK, W[0]), "a table"),
    (lambda: K.k_embedding(TOK, W[:, :0]), "a table"),
    (lambda: K.k_embedding(TOK.float(), W), "integer ids"),
    (lambda: K.k_embedding(TOK[:1, :1].expand(1 << 14, (1 << 13) + 1), W), "integer ids"),
    (lambda: K.k_embedding(TOK, W, padding_idx=16), "padding_idx"),
    (lambda: K.k_embedding(TOK, W, padding_idx=-1), "padding_idx"),
    (lambda: K.k_embedding(TOK.to("meta"), W), "must be on cpu"),
])
def test_arguments_are_refused_by_name(call, message):
    with pytest.raises(ValueError) as e:
        call()
    assert message in str(e.value), str(e.value)


@pytest.mark.parametrize("call", [lambda: K.k_token_logprobs(X, TOK, top_k=2), lambda: K.k_distill_topk(X, *LIST), lambda: K.k_embedding(TOK, W)])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="strict_cuda"):
        call()


# A pointer that nothing reads: every one of these calls is refused by the host before a launch.
P = C.c_void_p(4096)
BAD, ALIGN, CAPACITY = -1, -2, -7
SCORES = dict(logits=P, type=A.TYPE_BF16, ldl=64, tokens=P, ignore=-100, temperature=1.0, k=4, logprob=P, entropy=P, top=P, ids=P, stats=P, rows=2, V=64, status=None, stream=None)
SCORES_BWD = dict(logits=P, type=A.TYPE_BF16, ldl=64, tokens=P, temperature=1.0, k=4, ids=P, stats=P, entropy=P, g=P, gh=P, gt=P, dlogits=P, rows=2, V=64, stream=None)
DISTILL = dict(logits=P, type=A.TYPE_BF16, ldl=64, teacher=P, ids=P, k=4, temperature=1.0, tail=0, loss=P, stats=P, rows=2, V=64, status=None, stream=None)
DISTILL_BWD = dict(logits=P, type=A.TYPE_BF16, ldl=64, teacher=P, ids=P, k=4, temperature=1.0, stats=P, dloss=P, dlogits=P, rows=2, V=64, stream=None)
EMBED = dict(ids=P, n=4, table=P, type=A.TYPE_BF16, V=16, d=8, scale=1.0, out=P, status=None, stream=None)
EMBED_BWD = dict(ids=P, n=4, dy=P, type=A.TYPE_BF16, V=16, d=8, scale=1.0, padding=-1, dtable=P, scratch=P, bytes=1 << 20, status=None, stream=None)


@pytest.mark.parametrize("name, args, change, code", [
    *[("rte_token_logprobs_fwd", SCORES, {k: None}, BAD) for k in ("logits", "tokens", "logprob", "entropy", "top", "ids")],
    *[("rte_token_logprobs_fwd", SCORES, c, BAD) for c in ({"type": 3}, {"type": -1}, {"ldl": -1}, {"temperature": 0.0}, {"temperature": float("nan")}, {"k": -1},
                                                         {"k": 65}, {"k": 257, "V": 1000}, {"rows": 0}, {"rows": -5}, {"V": 0})],
    *[("rte_token_logprobs_bwd", SCORES_BWD, {k: None}, BAD) for k in ("logits", "tokens", "ids", "stats", "entropy", "dlogits")],
    *[("rte_token_logprobs_bwd", SCORES_BWD, c, BAD) for c in ({"type": 3}, {"ldl": -1}, {"temperature": -1.0}, {"k": 65}, {"rows": 0}, {"V": 0})],
    *[("rte_distill_topk_fwd", DISTILL, {k: None}, BAD) for k in ("logits", "teacher", "ids", "loss")],
    *[("rte_distill_topk_fwd", DISTILL, c, BAD) for c in ({"type": 3}, {"ldl": -1}, {"temperature": 0.0}, {"k": 0}, {"k": 257}, {"rows": 0}, {"V": 0})],
    ("rte_distill_topk_fwd", DISTILL, {"stats": C.c_void_p(4100)}, ALIGN),
    *[("rte_distill_topk_bwd", DISTILL_BWD, {k: None}, BAD) for k in ("logits", "teacher", "ids", "stats", "dloss", "dlogits")],
    *[("rte_distill_topk_bwd", DISTILL_BWD, c, BAD) for c in ({"type": 3}, {"temperature": 0.0}, {"k": 0}, {"rows": 0}, {"V": 0})],
    ("rte_distill_topk_bwd", DISTILL_BWD, {"stats": C.c_void_p(4104)}, ALIGN),
    *[("rte_embedding_fwd", EMBED, {k: None}, BAD) for k in ("ids", "table", "out")],
    *[("rte_embedding_fwd", EMBED, c, BAD) for c in ({"type": 3}, {"n": 0}, {"V": 0}, {"d": 0})],
    ("rte_embedding_fwd", EMBED, {"type": A.TYPE_F32, "table": C.c_void_p(4098)}, ALIGN),
    *[("rte_embedding_bwd", EMBED_BWD, {k: None}, BAD) for k in ("ids", "dy", "dtable", "scratch")],
    *[("rte_embedding_bwd", EMBED_BWD, c, BAD) for c in ({"type": 3}, {"n": 0}, {"n": (1 << 27) + 1}, {"V": 0}, {"V": 0x7FFFFFFF}, {"d": 0})],
    ("rte_embedding_bwd", EMBED_BWD, {"bytes": 16}, CAPACITY),
    ("rte_embedding_bwd", EMBED_BWD, {"scratch": C.c_void_p(4104)}, ALIGN),
    ("rte_embedding_bwd", EMBED_BWD, {"type": A.TYPE_F32, "dy": C.c_void_p(4098)}, ALIGN),
])
def test_the_c_abi_refuses_before_a_launch(name, args, change, code):
    assert getattr(A.load(), name)(*{**args, **change}.values()) == code


def test_scratch_of_the_embeddings_gradient_grows_with_the_call():
    need = A.load().rte_embedding_bwd_scratch
    assert need(0, 8) == 0 and need(5, 0) == 0 and need((1 << 27) + 1, 8) == 0
    assert 0 < need(1, 1) <= need(1, 1024) <= need(5000, 1024) < need(50000, 1024)
    assert need(1 << 27, 4096) > 1 << 32                  # (sizes of the largest call do not wrap)
