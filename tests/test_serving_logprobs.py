"""Log-probabilities of generated tokens: scheduler requests and /v1/completions."""
import json
import math

import pytest
import torch

from service_account_auth_improvements_amd.serving.engine import Request, Scheduler, build_engine, record_logprobs
from service_account_auth_improvements_amd.serving.server import create_app


@pytest.fixture(scope="module")
def eng():
    return build_engine("tiny", device="cpu", n_slots=4, max_len=64)


def _check_against_forward(eng, r, tol):
    """Each token's values against the whole sequence's forward pass (tol: the decode path's logit error)."""
    seq = torch.tensor([r.prompt + r.output])
    S = seq.shape[1]
    pad = (-S) % 128 if eng.dev.type == "cuda" else 0          # the forward's attention tiles
    seq = torch.nn.functional.pad(seq, (0, pad)).to(eng.dev)
    lp = torch.log_softmax(eng.m.forward_logits(seq)[0].float(), -1).cpu()
    assert len(r.token_logprobs) == len(r.output) == len(r.top_logprobs)
    for j, t in enumerate(r.output):
        row = lp[len(r.prompt) - 1 + j]
        assert abs(r.token_logprobs[j] - float(row[t])) < tol
        alts = r.top_logprobs[j]
        assert len(alts) == r.logprobs
        assert [v for _, v in alts] == sorted((v for _, v in alts), reverse=True)
        if alts:
            want = torch.topk(row, len(alts)).values
            assert (torch.tensor([v for _, v in alts]) - want).abs().max() < 2 * tol
            for i, v in alts:
                assert abs(v - float(row[i])) < tol
            if r.temperature == 0:
                assert alts[0] == (t, r.token_logprobs[j])


def test_scheduler_records_what_was_asked(eng):
    plain = Scheduler(eng, max_batch=4)
    ref = plain.submit(Request(prompt=[1, 2, 3], max_new_tokens=5))
    plain.run_until_idle()
    s = Scheduler(eng, max_batch=4)
    reqs = [Request(prompt=[1, 2, 3], max_new_tokens=5, logprobs=4), Request(prompt=[9, 8], max_new_tokens=6),
            Request(prompt=[4] * 7, max_new_tokens=3, logprobs=0), Request(prompt=[5, 6], max_new_tokens=4, temperature=0.8, logprobs=2)]
    for r in reqs:
        s.submit(r)
    s.run_until_idle()
    assert reqs[0].output == ref.output and not ref.token_logprobs and not ref.top_logprobs
    assert not reqs[1].token_logprobs and not reqs[1].top_logprobs
    for r in (reqs[0], reqs[2], reqs[3]):
        _check_against_forward(eng, r, 2e-2)


def test_out_of_range_is_refused(eng):
    s = Scheduler(eng, max_batch=2)
    for bad in (-1, 21):
        r = s.submit(Request(prompt=[1], max_new_tokens=2, logprobs=bad))
        assert r.done.is_set() and "logprobs" in r.error


def test_record_logprobs_small_vocabulary():
    logits = torch.tensor([[0.0, 1.0, 1.0], [2.0, float("-inf"), 0.0]])
    a, b = Request(prompt=[1], logprobs=20), Request(prompt=[1], logprobs=1)
    record_logprobs(logits, [2, 1], [a, b])
    assert [i for i, _ in a.top_logprobs[0]] == [1, 2, 0]           # equal logits by id
    assert b.token_logprobs == [float("-inf")] and b.top_logprobs[0][0][0] == 0


def test_completions_api(eng):
    s = Scheduler(eng, max_batch=4).start()
    try:
        app = create_app(s, "llama").test_client()
        base = app.post("/v1/completions", json={"prompt": "hello", "max_tokens": 3}).json
        assert "logprobs" not in base["choices"][0]
        r = app.post("/v1/completions", json={"prompt": ["hello", "a"], "max_tokens": 3, "logprobs": 3})
        for c in r.json["choices"]:
            lp = c["logprobs"]
            assert len(lp["tokens"]) == len(lp["token_logprobs"]) == len(lp["top_logprobs"]) == len(lp["text_offset"]) == 3
            assert all(v <= 0 and math.isfinite(v) for v in lp["token_logprobs"])
            assert all(len(d) == 3 and max(d.values()) == pytest.approx(v) for d, v in zip(lp["top_logprobs"], lp["token_logprobs"]))
            assert lp["text_offset"][0] == 0 and "".join(lp["tokens"])[:lp["text_offset"][2]] == "".join(lp["tokens"][:2])
        assert r.json["choices"][0]["token_ids"] == base["choices"][0]["token_ids"]
        zero = app.post("/v1/completions", json={"prompt": "a", "max_tokens": 2, "logprobs": 0}).json["choices"][0]["logprobs"]
        assert zero["top_logprobs"] is None and len(zero["token_logprobs"]) == 2
        none = app.post("/v1/completions", json={"prompt": "a", "max_tokens": 2, "logprobs": None}).json["choices"][0]
        assert "logprobs" not in none
        json.loads(r.get_data(as_text=True), parse_constant=lambda c: pytest.fail(c))     # no NaN / Infinity
        for bad in (-1, 21, 1.5, "3", True):
            assert app.post("/v1/completions", json={"prompt": "a", "max_tokens": 2, "logprobs": bad}).status_code == 400
    finally:
        s.stop()


@pytest.mark.gpu
def test_scheduler_records_on_the_gpu():
    eng = build_engine("small", device="cuda:0", n_slots=6, max_len=256, n_layers=2)
    s = Scheduler(eng, max_batch=6)
    reqs = [Request(prompt=list(range(3, 3 + 5 * n)), max_new_tokens=6, logprobs=n, temperature=0.0 if n != 3 else 0.7)
            for n in (1, 2, 3, 20)] + [Request(prompt=[7, 8], max_new_tokens=6)]
    for r in reqs:
        s.submit(r)
    s.run_until_idle()
    assert not reqs[-1].token_logprobs
    for r in reqs[:-1]:
        _check_against_forward(eng, r, 5e-2)


class _Written:
    """A scheduler that answers every request with given tokens."""

    e = None

    def __init__(self, output):
        self.output = output

    def submit(self, r):
        r.output = list(self.output)
        r.token_logprobs = [-1.0] * len(r.output)
        r.top_logprobs = [[(t, -1.0)] for t in r.output]
        r.t_submit = r.t_first = 0.0
        r.done.set()
        return r


class _SpaceTokenizer:
    """Words with a space before each but the first of what is decoded, as sentence-piece vocabularies are."""

    def encode(self, text):
        return [len(w) for w in text.split()]

    def decode(self, ids):
        return " ".join("w" * i for i in ids)


@pytest.mark.parametrize("text", ["é!", "aé漢😀b", "", "plain", "😀😀"])
def test_text_offsets_lie_in_the_text(text):
    """A token's offset is where its first character starts; the bytes of one character share theirs."""
    app = create_app(_Written(text.encode()), "m").test_client()
    c = app.post("/v1/completions", json={"prompt": "a", "max_tokens": 4, "logprobs": 1}).json["choices"][0]
    assert c["text"] == text
    want = [i for i, ch in enumerate(text) for _ in ch.encode()]
    assert c["logprobs"]["text_offset"] == want


def test_text_offsets_of_bytes_that_are_no_text():
    # two bytes of no character, one, two that start a character which never ends, one, 900 as the first
    out = [255, 254, 65, 0xE2, 0x82, 66] + [255] * 900 + [67]
    app = create_app(_Written(out), "m").test_client()
    c = app.post("/v1/completions", json={"prompt": "a", "max_tokens": 4, "logprobs": 0}).json["choices"][0]
    assert c["text"] == "��A�B" + "�" * 900 + "C"
    off = c["logprobs"]["text_offset"]
    assert off[:4] == [0, 1, 2, 3] and off[4] in (3, 4) and off[5:] == list(range(4, 4 + 902))


def test_text_offsets_where_a_first_space_is_dropped():
    app = create_app(_Written([3, 1, 4, 1, 5]), "m", tokenizer=_SpaceTokenizer()).test_client()
    c = app.post("/v1/completions", json={"prompt": "a", "max_tokens": 4, "logprobs": 1}).json["choices"][0]
    off = c["logprobs"]["text_offset"]
    assert [c["text"][a:b].strip() for a, b in zip(off, off[1:] + [None])] == ["www", "w", "wwww", "w", "wwwww"]
