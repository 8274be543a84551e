"""GPU: BatchedTTSDecoder(mode="paged") -- plans, stores and attention over the page pool inside the whole backbone --
against the CPU oracle's transformers bf16 policy (the prefill's own bar, rel-L2 1e-2: bf16 storage after every
op, f32 sums in another order), its sampler on the GPU's logits, and itself."""
import pytest
import torch

from oracle.qtts_oracle import DecoderOracle, TalkerWeights, apply_repetition_penalty, head_logits, rel_l2, sample_token, suppress_mask

pytestmark = pytest.mark.gpu
TOL = 1e-2
EOS = 2150
LENS = [5, 40, 1, 17, 64, 33, 2, 16, 65, 9, 31]          # 11 streams: more than one launch of the other modes


@pytest.fixture(scope="module")
def model(pkg):
    sd = pkg.synthetic_state_dict(seed=21, cfg=pkg.SyntheticConfig(n_bb_layers=2, n_cp_layers=1, n_groups=15))
    return {k: v.cuda() for k, v in sd.items()}, TalkerWeights.from_state_dict(sd, 2, 1)


def rows(seed, n):
    return torch.randn(n, 1024, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


def oracle_run(tw, xs):
    orc = DecoderOracle(tw.bb_layers, tw.bb_norm, 128, "backbone", "hf_bf16")
    return [orc.step(x, pos=i)[0] for i, x in enumerate(xs)], orc


@pytest.mark.parametrize("page_size", [16, 64])
def test_prompts_and_steps_match_the_oracle(pkg, model, page_size):
    """Ragged prompts in one call, two steps, a prompt piece appended to some streams, a last step; the pool's K and V."""
    dsd, tw = model
    n = len(LENS)
    dec = pkg.BatchedTTSDecoder(dsd, n, max_seq_len=128, mode="paged", page_size=page_size)
    xs = [rows(100 + s, LENS[s] + 13) for s in range(n)]
    refs, orcs = zip(*[oracle_run(tw, xs[s][:LENS[s] + 13]) for s in range(n)])
    at = [0] * n

    def feed(counts):
        packed = torch.cat([xs[s][at[s]:at[s] + c] for s, c in enumerate(counts)]).cuda()
        h = dec.paged.forward(packed, counts)
        for s, c in enumerate(counts):
            at[s] += c
            if c:
                assert rel_l2(h[s].cpu(), refs[s][at[s] - 1]) < TOL, (s, at[s])
            else:
                assert bool((h[s] == 0).all())

    feed(LENS)
    feed([1] * n)
    tok = torch.zeros(n, dtype=torch.int32, device="cuda")
    h = dec.step_select(torch.stack([xs[s][at[s]] for s in range(n)]).cuda(), tok, EOS)
    for s in range(n):
        at[s] += 1
        assert rel_l2(h[s].cpu(), refs[s][at[s] - 1]) < TOL
    feed([10 if s % 3 == 0 else 0 for s in range(n)])
    feed([1] * n)
    dec.check_error()
    assert dec.positions() == at and dec.paged.lengths.tolist() == at
    table = dec.paged.block_table.cpu()
    for s in range(n):
        page = table[s, :-(-at[s] // page_size)].long()
        for pool, want in ((dec.paged.k_pool, orcs[s].k), (dec.paged.v_pool, orcs[s].v)):
            got = pool[:, page].permute(0, 2, 1, 3, 4).reshape(2, 8, -1, 128)[:, :, :at[s]]
            assert rel_l2(got.float().cpu(), want[:, :, :at[s]].float()) < TOL


def test_matches_the_prefill_kernel(pkg, model):
    """One long prompt through the pool and through qtts_backbone_prefill (the same projections)."""
    dsd, _ = model
    x = rows(3, 700).cuda()
    one = pkg.TTSMegakernelGenerator(model=dsd, max_seq_len=1024)
    h1 = one.prefill(x)
    dec = pkg.BatchedTTSDecoder(dsd, 2, max_seq_len=1024, mode="paged")
    h2 = dec.paged.forward(torch.cat([x, x[:30]]), [700, 30])
    assert rel_l2(h2[0].cpu(), h1.cpu()) < TOL
    dec.set_kv_cache(1, one.get_k_cache()[:, :, :700], one.get_v_cache()[:, :, :700])      # the contiguous cache's K and V
    assert dec.positions() == [700, 700]
    step = torch.cat([x[:1], x[:1]])
    h3 = dec.paged.forward(step, [1, 1])
    assert rel_l2(h3[0].cpu(), h3[1].cpu()) < TOL


@pytest.mark.parametrize("sample", [False, True])
def test_selection_matches_the_oracle_sampler(pkg, model, sample):
    dsd, tw = model
    n = 9
    dec = pkg.BatchedTTSDecoder(dsd, n, max_seq_len=64, mode="paged")
    i32 = dict(dtype=torch.int32, device="cuda")
    tok, logits = torch.full((n,), -7, **i32), torch.zeros(n, 3072, device="cuda")
    hist = torch.randint(0, 2200, (n, 20), generator=torch.Generator().manual_seed(4)).to(torch.int32).cuda()
    hist[0, :2] = torch.tensor([-5, 9999], **i32)              # ids outside the head penalise nothing
    nh = [2, 0, 20, 7, 7, 1, 3, 20, 5]
    skip = torch.tensor([0, 0, 1, 0, 0, 0, 0, 1, 0], **i32)
    kw = dict(do_sample=sample, temperature=0.9, top_k=50, top_p=0.9, seed=31, frame_step=4)
    h = dec.paged.forward(rows(8, n).cuda(), [1] * n, tok, skip, history=hist, n_history=torch.tensor(nh, **i32), history_len=0,
                          repetition_penalty=1.3, eos_id=EOS, suppress_eos=True, out_logits=logits, **kw)
    for s in range(n):
        if skip[s]:
            assert tok[s] == -7 and bool((h[s] == 0).all()) and bool((logits[s] == 0).all())
            continue
        lg = logits[s].cpu()
        # one bf16 step of the logit: the head's f32 sums against f64
        assert bool(((lg - head_logits(tw.codec_head, h[s])).abs() <= 2.0 ** -7 * lg.abs() + 1e-4).all())
        lg = apply_repetition_penalty(lg, [i for i in hist[s, :nh[s]].tolist() if 0 <= i < 3072], 1.3)
        lg[suppress_mask(3072, EOS)] = float("-inf")
        assert int(tok[s]) == sample_token(lg, sample, 0.9, 50, 0.9, EOS, seed=31 + s, frame_step=4, group=0)
    # skipped streams' positions advance all the same, but they hold nothing for it
    assert dec.positions() == [1] * n and dec.paged.lengths.tolist() == (1 - skip).tolist()


@pytest.mark.parametrize("sample", [False, True], ids=["greedy", "sampled"])
def test_generate(pkg, model, sample):
    """11 utterances in one batch; the EOS id is one that stream 0 chooses at a frame k: it ends there, and every other
    stream runs on as before until it chooses the id itself."""
    dsd, _ = model
    n, most = len(LENS), 14
    prompts = [rows(200 + s, LENS[s])[None] for s in range(n)]
    texts = [rows(300 + s, 1 + s % 4)[None] for s in range(n)]
    pad = rows(9, 1)[None]
    kw = dict(do_sample=sample, temperature=0.9, top_k=40, top_p=0.9, cp_do_sample=sample, cp_top_k=30, repetition_penalty=1.1,
              seed=5, sync_every=4)
    dec = pkg.BatchedTTSDecoder(dsd, n, max_seq_len=96, mode="paged", page_size=16)
    free = dec.generate(prompts, texts, pad, 3000, max_tokens=most, min_new_tokens=most, **kw)
    assert [len(f) for f in free] == [most] * n
    g0 = [f[0] for f in free[0]]
    k = next(i for i in range(4, most) if g0[i] not in g0[:i])
    out = dec.generate(prompts, texts, pad, g0[k], max_tokens=most, min_new_tokens=2, **kw)
    for s in range(n):
        ids = [f[0] for f in free[s]]
        end = next((i for i, t in enumerate(ids) if t == g0[k]), most)
        assert out[s] == free[s][:end] or g0[k] in ids[:2], s
    assert out[0] == free[0][:k]


def test_window_bounds_what_a_token_attends(pkg, model):
    """Under a window and sinks the K and V of the keys between them do not matter."""
    dsd, _ = model
    x = rows(11, 90).cuda()
    hs = []
    for noise in (0.0, 50.0):
        dec = pkg.BatchedTTSDecoder(dsd, 1, max_seq_len=128, mode="paged", page_size=16, window=20, sinks=3)
        dec.paged.forward(x, [90])
        for pool in (dec.paged.k_pool, dec.paged.v_pool):       # tokens 16 .. 63: past the sinks, before the window
            pool[:, dec.paged.block_table[0, 1:4].long()] += noise
        hs.append(dec.paged.forward(x[:1], [1]))
    assert torch.equal(hs[0], hs[1])
    full = pkg.BatchedTTSDecoder(dsd, 1, max_seq_len=128, mode="paged", page_size=16)
    full.paged.forward(x, [90])
    assert rel_l2(full.paged.forward(x[:1], [1]).cpu(), hs[0].cpu()) > TOL


def test_pool_runs_out_and_is_reset(pkg, model):
    dsd, _ = model
    dec = pkg.BatchedTTSDecoder(dsd, 3, max_seq_len=64, mode="paged", page_size=16, num_pages=5)
    dec.paged.forward(rows(1, 32 + 16 + 16).cuda(), [32, 16, 16])
    dec.check_error()
    tok = torch.zeros(3, dtype=torch.int32, device="cuda")
    dec.step_select(rows(2, 3).cuda(), tok, EOS)                # three more pages asked for, one is there
    with pytest.raises(RuntimeError, match=r"streams \[1, 2\]"):
        dec.check_error()
    assert dec.paged.lengths.tolist() == [33, 16, 16]
    dec.paged.reset([1, 2])
    dec.check_error()
    assert dec.paged.free_count.item() == 2
    h = dec.paged.forward(rows(3, 1 + 8 + 8).cuda(), [1, 8, 8])
    dec.check_error()
    assert torch.isfinite(h).all() and dec.positions() == [34, 8, 8]


def test_finished_streams_take_no_pages(pkg, model):
    """Steps with ``skip``: the pool's last pages go to the streams that go on, whose results are those of a decoder
    without the finished ones; a finished stream is no failure."""
    dsd, _ = model
    make = lambda n, pages: pkg.BatchedTTSDecoder(dsd, n, max_seq_len=64, mode="paged", page_size=16, num_pages=pages)
    dec, alone = make(4, 6), make(2, 4)
    x = rows(1, 64).cuda()
    dec.paged.forward(x, [16] * 4)
    alone.paged.forward(torch.cat((x[16:32], x[48:])), [16, 16])
    skip = torch.tensor([1, 0, 1, 0], dtype=torch.int32, device="cuda")
    tok, tok2 = torch.full((4,), -7, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for i in range(3):
        y = rows(5 + i, 4).cuda()
        h = dec.step_select(y, tok, EOS, skip=skip)
        h2 = alone.step_select(y[1::2].contiguous(), tok2, EOS)
        assert torch.equal(h[1::2], h2) and bool((h[::2] == 0).all())
        assert torch.equal(tok[1::2], tok2) and tok[::2].tolist() == [-7, -7]
    dec.check_error()
    assert dec.paged.lengths.tolist() == [16, 19, 16, 19] and dec.paged.free_count.item() == 0


def test_refused_calls_leave_the_pool_as_it_was(pkg, model):
    dsd, _ = model
    dec = pkg.BatchedTTSDecoder(dsd, 2, max_seq_len=64, mode="paged", page_size=16, num_pages=3)
    x, ok = rows(1, 2).cuda(), torch.zeros(2, dtype=torch.int32, device="cuda")
    for call in (lambda: dec.step_select(x, ok.cpu(), EOS), lambda: dec.step_select(x, torch.zeros(2, 2, dtype=torch.int32, device="cuda")[:, 0], EOS),
                 lambda: dec.step_select(x, ok, EOS, skip=ok.cpu()), lambda: dec.step_select(x, ok, EOS, do_sample=True, temperature=0.0),
                 lambda: dec.paged.forward(x, [1]), lambda: dec.paged.forward(x, [3, -1]), lambda: dec.paged.forward(x[:0], [0, 0])):
        with pytest.raises(ValueError):
            call()
    k = torch.zeros(2, 8, 64, 128)
    with pytest.raises(RuntimeError, match="free pages"):
        dec.set_kv_cache(1, k, k)
    assert dec.positions() == [0, 0] and dec.paged.lengths.tolist() == [0, 0] and dec.paged.free_count.item() == 3
    dec.check_error()
    # other types and strides of embeddings are taken as they are
    a = dec.paged.forward(x, [1, 1])
    dec.paged.reset()
    b = dec.paged.forward(x.float().t().contiguous().t(), [1, 1])
    assert torch.equal(a, b)


def test_refusals(pkg, model):
    dsd, _ = model
    with pytest.raises(ValueError, match="page_size"):
        pkg.BatchedTTSDecoder(dsd, 1, mode="paged", page_size=48)
    with pytest.raises(ValueError, match="mode='paged'"):
        pkg.BatchedTTSDecoder(dsd, 1, window=5)
    dec = pkg.BatchedTTSDecoder(dsd, 2, max_seq_len=32, mode="paged")
    with pytest.raises(RuntimeError, match="max_seq_len"):
        dec.paged.forward(rows(1, 34).cuda(), [33, 1])
    with pytest.raises(ValueError, match="embeds"):
        dec.paged.forward(rows(1, 3).cuda(), [1, 1])
    with pytest.raises(ValueError, match="n_history"):
        dec.step_select(rows(1, 2).cuda(), torch.zeros(2, dtype=torch.int32, device="cuda"), EOS, torch.zeros(2, 4, dtype=torch.int32), [5, 0])
    with pytest.raises(ValueError, match="k and v"):
        dec.set_kv_cache(0, torch.zeros(2, 8, 4, 64), torch.zeros(2, 8, 4, 64))
    with pytest.raises(ValueError, match="mfma"):
        dec.generate([rows(1, 2)[None]] * 2, [rows(1, 2)[None]] * 2, rows(1, 1)[None], EOS, max_tokens=3, prefill="steps")
    assert dec.positions() == [0, 0] and dec.paged.lengths.tolist() == [0, 0]
