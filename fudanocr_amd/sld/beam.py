"""Beam search with the transformer recognizers (sld.model.transformer, loss.transformer and loss.transformer_english_decomposition:
one decoder block each): every step runs the decoder on the beams' newest tokens alone.  The keys and values of the earlier
ones lie in a paged cache (fudanocr_amd/decode.py) that is reordered with the surviving beams, those of the image's positions
are computed once and read by all of an image's beams together.

Without it, the models answer by running the whole prefix through the decoder again for every token and taking the best one;
`beams=1` gives the same strings."""
import torch

from .. import kernels as K
from ..decode import PagedCache, beam_select


def _norm(ln, x, residual):
    a, b = (ln.a, ln.b) if hasattr(ln, "a") else (ln.a_2, ln.b_2)
    return K.layernorm_std(x, a, b, residual=residual, eps=ln.eps)


@torch.no_grad()
def search(model, batch, encode, embedding, generator, beams, max_len, start, eos):
    """encode() -> the encoder's output NHWC [batch, H, W, 1024], called once the arguments are checked -> (tokens
    int64 [batch, beams, max_len], scores fp32 [batch, beams]), best first.  A hypothesis ends with its first `eos`; the
    positions behind it hold `eos` too.  Nothing in here waits for the device."""
    if model.training:
        raise RuntimeError("beam_search needs the model in eval mode")
    if not (1 <= beams <= 64 and max_len >= 1 and max_len <= model.pe.pe.shape[1]):
        raise RuntimeError("beam_search: beams must be 1 to 64, max_len 1 to %d" % model.pe.pe.shape[1])
    if batch * beams > 65535 and max_len > 1:               # (a single step reorders nothing)
        raise RuntimeError("beam_search: batch x beams must be at most 65535, got %d x %d" % (batch, beams))
    vocab = generator.proj.weight.shape[0]
    if not (0 <= start < vocab and 0 <= eos < vocab):
        raise RuntimeError("beam_search: start and eos must be inside the %d classes" % vocab)
    feat = encode()
    dec, dev = model.decoder, feat.device
    own, cross = dec.mask_multihead, dec.multihead
    _, hh, ww, dm = feat.shape
    slots = batch * beams
    if batch == 0:
        return torch.empty((0, beams, max_len), dtype=torch.int64, device=dev), torch.empty((0, beams), device=dev)

    def heads(x, mha):
        return x.view(-1, mha.h, mha.d_k)

    mem = feat.reshape(batch, hh * ww, dm)
    image = PagedCache(batch, hh * ww, cross.h, cross.d_k, page=64, device=dev)
    image.advance(hh * ww)
    image.append(0, heads(cross.linears[1](mem), cross), heads(cross.linears[2](mem), cross))
    cache = PagedCache(slots, max_len, own.h, own.d_k, page=16, device=dev)
    token = torch.full((slots,), start, dtype=torch.int64, device=dev)
    scores = torch.full((batch, beams), float("-inf"), device=dev)
    scores[:, 0] = 0.0                                      # the beams differ from the second step on
    finished = torch.zeros((batch, beams), dtype=torch.bool, device=dev)
    history = []
    for t in range(max_len):
        emb = embedding(token)                              # [slots, 512]
        pos = model.pe.pe[0, t].expand(slots, -1).contiguous()
        x = K.concat_pe(emb.view(1, slots, -1), pos).view(slots, 1, dm)
        q, k, v = (heads(lin(x), own) for lin in own.linears[:3])
        cache.advance(1)
        cache.append(0, k, v)
        r = _norm(dec.mul_layernorm1, own.linears[3](cache.attend(0, q).view(slots, 1, dm)), x)
        # an image's beams are the rows of one chunk: its keys and values are read once for all of them
        a = image.attend(0, heads(cross.linears[0](r), cross), causal=False)
        r = _norm(dec.mul_layernorm2, cross.linears[3](a.view(slots, 1, dm)), r)
        r = _norm(dec.mul_layernorm3, dec.pff(r), r)
        logits = generator(r).view(batch, beams, vocab)
        scores, parents, tokens, finished = beam_select(logits, scores, finished, eos=eos)
        history.append((parents, tokens))
        if t + 1 < max_len:
            cache.reorder(parents)
            token = tokens.view(slots)
    out = torch.empty((batch, beams, max_len), dtype=torch.int64, device=dev)
    at = torch.arange(beams, device=dev).expand(batch, beams)
    for t in range(max_len - 1, -1, -1):                    # back from the survivors to their first tokens
        parents, tokens = history[t]
        out[:, :, t] = torch.gather(tokens, 1, at)
        at = torch.gather(parents, 1, at).long()
    return out, scores
