"""Models with the 4-bit KV cache (kv_type q4_0) and with a window and sinks, through the C ABI:

- logits against a float64 forward pass that keeps K and V as the cache holds them (Granite without scales is the llama
  layer, OLMo 2 the one with whole-row norms and NEOX pairs; token by token, and as one prompt);
- ForwardBatch rows bit-identical to single steps; sequences that grow, truncate and stream the same as ones that do not;
- a serving run: a batch of prompts, then steps sampled with every filter, append, attention and sampler together.

A logit may differ from the float64 pass's by more than fp32 noise, because a key or value that lies at a code's border
takes the other code: activations are off by 1e-4 of their size at most, a code's step is about a quarter of it, so one code in
a thousand may flip, by a quarter: sqrt(1e-3) / 4 < 1% of the keys' and values' size, where rounding them to 4 bits
itself is about 8%. The bound is 3% of the logits' spread, and the fp16 cache's logits lie outside it."""
import numpy as np
import pytest

import kv4_ref as R
from naive_arch import NaiveArch
from test_gpu_sample_rows import DT, reference
from windlass_b200 import _lib
from windlass_b200.transformer import CudaTransformer, config0_spec, synth_spec

pytestmark = pytest.mark.gpu

Q4 = _lib.TYPES["q4_0"]
PROBE = [1, 10, 50, 100, 200, 257, 290, 5, 7, 99, 33, 72, 12, 13, 14, 15, 16, 17, 18, 19]


def held(v, hd):
    c, d = R.quantise(np.asarray(v, np.float64).reshape(-1, hd))
    return ((c - 8) * np.repeat(d.astype(np.float64), 32, -1)).reshape(-1)


class NaiveKv4(NaiveArch):
    """NaiveArch with the K and V rows as the 4-bit cache holds them, and a window with sinks."""

    def __init__(self, *a, window=0, sinks=0, **kw):
        super().__init__(*a, **kw)
        self.window, self.sinks = window, sinks

    def forward(self, toks):
        n, W = self.n, self.n.W
        olmo = self.arch == "olmo2"
        H, KV, HD = self.H, self.KV, self.HD
        embd, head = W("token_embd.weight"), W("output.weight")
        K, V, out = [[] for _ in range(self.L)], [[] for _ in range(self.L)], []
        for t, tok in enumerate(toks):
            x = embd[tok] * self.es
            see = R.visible(t, self.window, self.sinks)
            for l in range(self.L):
                p = f"blk.{l}."
                h = x if olmo else n.rms(x, W(p + "attn_norm.weight"))
                q, k, v = W(p + "attn_q.weight") @ h, W(p + "attn_k.weight") @ h, W(p + "attn_v.weight") @ h
                if olmo:
                    q, k = n.rms(q, W(p + "attn_q_norm.weight")), n.rms(k, W(p + "attn_k_norm.weight"))
                for hh in range(H):
                    self.rope(q, hh * HD, HD, t, 500000.0, olmo)
                for hh in range(KV):
                    self.rope(k, hh * HD, HD, t, 500000.0, olmo)
                K[l].append(held(k, HD))
                V[l].append(held(v, HD))
                Kl, Vl, att = np.stack(K[l])[see], np.stack(V[l])[see], np.zeros(H * HD)
                for hh in range(H):
                    c = slice(hh // (H // KV) * HD, (hh // (H // KV) + 1) * HD)
                    s = Kl[:, c] @ q[hh * HD:(hh + 1) * HD] * self.kq
                    e = np.exp(s - s.max())
                    att[hh * HD:(hh + 1) * HD] = (e / e.sum()) @ Vl[:, c]
                o = W(p + "attn_output.weight") @ att
                x = x + (n.rms(o, W(p + "post_attention_norm.weight")) if olmo else o) * self.rs
                f = n.swiglu(W(p + "ffn_gate.weight"), W(p + "ffn_up.weight"), W(p + "ffn_down.weight"), x if olmo else n.rms(x, W(p + "ffn_norm.weight")))
                x = x + (n.rms(f, W(p + "post_ffw_norm.weight")) if olmo else f) * self.rs
            out.append(head @ n.rms(x, W("output_norm.weight")) / self.div)
        return np.stack(out)


@pytest.mark.parametrize("arch", ["granite", "olmo2"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (5, 2)])
def test_logits_of_a_float64_pass_over_the_held_values(wl, oracle, tmp_path, arch, window, sinks):
    O = oracle
    p = O.write_tiny_arch(str(tmp_path / f"{arch}.gguf"), arch, O.Q8_0)
    ref = NaiveKv4(O, p, arch, window=window, sinks=sinks)
    want = ref.forward(PROBE)
    ref.close()
    std = want.std()
    with CudaTransformer(p, max_context=512, kv_type=Q4, attn_window=window, attn_sinks=sinks) as m:
        whole = m.forward(PROBE, all_logits=True)
        m.truncate(0)
        steps = np.stack([m.forward([t], pos0=i) for i, t in enumerate(PROBE)])
        m.truncate(7)
        tail = m.forward(PROBE[7:], pos0=7, all_logits=True)
    for got in (whole, steps, tail):
        assert np.abs(got - want[-len(got):]).max() < 0.03 * std, np.abs(got - want[-len(got):]).max() / std
    with CudaTransformer(p, max_context=512) as m:
        fp16 = m.forward(PROBE, all_logits=True)
    assert np.abs(fp16 - want).max() > 0.03 * std


@pytest.mark.parametrize("spec", [config0_spec(), synth_spec("qwen3moe", 2, 256, 16, 2, 128, 0, 2048, 4096, experts=8, experts_used=2,
                                                             expert_ff=256, rms_eps=1e-6, type_embd=12)], ids=["llama", "qwen3moe"])
@pytest.mark.parametrize("window", [0, 24])
def test_batch_rows_are_bit_identical_to_single_steps(wl, spec, window):
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 2000, n).astype(np.int32) for n in (3, 40, 1, 17, 9)]
    kw = dict(synthetic=spec, max_context=256, kv_type=Q4, attn_window=window, attn_sinks=4 if window else 0)
    with CudaTransformer(**kw) as m, CudaTransformer(**kw) as solo:
        seqs, ref = [m.new_sequence() for _ in prompts], [solo.new_sequence() for _ in prompts]
        for s, r, pr in zip(seqs, ref, prompts):
            m.forward(pr, seq=s)
            solo.forward(pr, seq=r)
        toks = rng.integers(0, 2000, len(prompts)).astype(np.int32)
        for step in range(3):
            rows = m.forward_batch(seqs, toks)
            for i in range(len(prompts)):
                one = solo.forward([toks[i]], pos0=ref[i].length, seq=ref[i])
                assert np.array_equal(rows[i].view(np.uint32), one.view(np.uint32)), (step, i)
            toks = rows.argmax(1).astype(np.int32)


def test_growing_and_streamed_sequences_keep_their_bits(wl):
    rng = np.random.default_rng(5)
    prompt = rng.integers(0, 4096, 250).astype(np.int32)
    kw = dict(synthetic=config0_spec(), max_context=1024, kv_type=Q4)
    with CudaTransformer(**kw) as a, CudaTransformer(**kw, use_graphs=0) as b, CudaTransformer(**kw, resident=0) as c:
        tok = int(np.argmax(a.forward(prompt)))
        b.forward(prompt)
        c.forward(prompt)
        ids = a.generate_greedy(tok, 30)                # room for all 30 at once
        t, got, streamed = tok, [], []
        for i in range(30):                             # step by step, past the first 256 positions' room
            lg = b.forward([t], pos0=250 + i)
            lc = c.forward([t], pos0=250 + i)
            assert np.array_equal(lg.view(np.uint32), lc.view(np.uint32)), i
            t = int(np.argmax(lg))
            got.append(t)
        assert got == list(ids)


def test_prompts_of_any_length_have_the_workspace_they_need(wl):
    """The ranges that a prompt is cut into, and so what its partial results take, do not fall steadily with its length (64
    heads on 8, a cache of 2048: 193 rows need none, 289 more than all shorter ones)."""
    rng = np.random.default_rng(7)
    spec = synth_spec("llama", 1, 256, 64, 8, 64, 256, 1024, 2048, rope_base=10000.0, type_ffn_down=8, seed=1)
    with CudaTransformer(synthetic=spec, max_context=2048, kv_type=Q4) as m:
        for n in (193, 289, 400):
            prompt = rng.integers(0, 1024, n).astype(np.int32)
            a, b = m.new_sequence(), m.new_sequence()
            one = m.forward(prompt, seq=a)
            for i in range(0, n, 97):
                parts = m.forward(prompt[i:i + 97], pos0=i, seq=b)
            # (as in the mixed steps below: two paths' flips)
            assert np.abs(one - parts).max() < 0.058 * one.std(), n


def test_mixed_steps_and_a_sampled_serving_run(wl):
    """Prompts of many lengths join in mixed steps, then a batch decodes with every row's own sampling options: each id is
    the sampler's choice on that row's own logits, taken from a model that runs the row alone."""
    rng = np.random.default_rng(11)
    kw = dict(synthetic=config0_spec(), max_context=512, kv_type=Q4, attn_window=128, attn_sinks=4)
    with CudaTransformer(**kw) as m, CudaTransformer(**kw) as solo:
        lists = [rng.integers(0, 4096, n).astype(np.int32) for n in (150, 3, 1, 40, 9, 2)]
        seqs, ref = [m.new_sequence() for _ in lists], [solo.new_sequence() for _ in lists]
        mixed = m.forward_mixed(seqs, lists)
        for i, (r, pr) in enumerate(zip(ref, lists)):
            one = solo.forward(pr, seq=r)
            # two paths (the tensor-core GEMM here, the matvec there), each with its own flips of 1% of the size: together
            # sqrt(2) * 1% of the spread, and the largest of 4096 logits lies sqrt(2 ln 4096) = 4.1 of that out: 5.8%
            assert np.abs(mixed[i] - one).max() < 0.058 * one.std(), i
        assert [s.length for s in seqs] == [len(x) for x in lists]
        # (the prompts took different paths, so that codes at a border may differ: continue from the same caches)
        n = len(lists)
        for s, r, pr in zip(seqs, ref, lists):
            s.truncate(0)
            m.forward(pr, seq=s)
        toks = rng.integers(0, 4096, n).astype(np.int32)
        for step in range(6):
            o = np.zeros(n, DT)
            o["temperature"], o["draw"] = rng.choice([0.0, 0.7, 1.2], n), rng.random(n)
            o["top_k"], o["top_p"], o["min_p"] = rng.choice([0, 40], n), rng.choice([1.0, 0.9], n), rng.choice([0.0, 0.02], n)
            got = m.forward_batch_sample_opts(seqs, toks, o["draw"], o["temperature"], o["top_k"], o["top_p"], o["min_p"])
            for i in range(n):
                lg = solo.forward([toks[i]], pos0=ref[i].length, seq=ref[i])
                want, margin = reference(lg, o[i])
                assert got[i] == want or margin < 1e-11, (step, i)
            toks = got.copy()


def test_decode_bench_and_profile_run(wl):
    with CudaTransformer(synthetic=config0_spec(), max_context=512, kv_type=Q4) as m:
        s = [m.new_sequence() for _ in range(3)]
        assert m.bench_decode(s, 5) > 0 and [x.length for x in s] == [5, 5, 5]
        m.profile(True)
        m.forward([1, 2, 3])
        assert m.profile_get(40).launches == 4 and m.profile_get(42).launches == 4
