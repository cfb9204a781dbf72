"""Evaluation on MI355X: full-graph student embedding, edge scoring and
Hits@K / AUC on the device.

Reference: ``test_transductive`` (src/train_teacher_gnn.py:76-155) and
``test_production`` (src/train_teacher_gnn.py:157-268); metrics are ogb 1.3.6
``Evaluator`` hits@K and sklearn ``roc_auc_score``.  The result dictionaries
have the reference's keys and tuple layouts, so ``logger.py`` and the
printing code of ``main.py`` consume them unchanged.

Scores are computed by ``EdgeScorer``: the predictor's first GEMM reads
``h[e0] * h[e1]`` through a gathered operand (no materialised pair tensor),
hidden layers keep bias+ReLU in the epilogue, and the Linear(H,1)+sigmoid
head is one reduction kernel.  Chunks of ``chunk`` edges bound the scratch.

dtype "mxfp4": the student answers in 4 bits (llp_mx).  Node features, pair products and hidden
activations are quantised (a hidden layer hands MXFP4 rows to the next), weights too; embeddings are
bf16 and the Linear(H, 1) head works on the last hidden layer in bf16.
Every call quantises the weights anew, so MXFP4 pays for many edges or nodes: 262,144 edges of 1,024-wide embeddings through
one hidden layer 0.90 ms (bf16 1.44), two 1.08 (1.87), two of 2,048 2.6 (5.9); one edge at width 256 53 us (bf16 43).
"""
from __future__ import annotations

import torch

import llp_hip as K
import llp_mx

TRANSDUCTIVE_KS = (10, 20, 30, 50)          # src/train_teacher_gnn.py:118
COLLAB_KS = (10, 50, 100)                   # src/train_teacher_gnn.py:132


def _as_pairs(edges: torch.Tensor) -> torch.Tensor:
    """[E, 2] int32 contiguous on the device (the reference keeps [E, 2])."""
    if edges.dim() != 2 or edges.shape[1] != 2:
        raise ValueError("edges must be [E, 2]")
    return edges.to(torch.int32).contiguous()


def _mx_weight(lin):
    """A layer's weight in MXFP4 (through f32 where it is in another type than f32 / bf16)."""
    w = lin.weight.detach()
    return llp_mx.quantize((w if w.dtype in (torch.float32, torch.bfloat16) else w.float()).contiguous())


class EdgeScorer:
    """predictor(h[e0], h[e1]) (src/models.py:139-150) in eval mode."""

    def __init__(self, predictor, dtype=torch.float32, chunk: int = 1 << 18):
        self.predictor = predictor
        self.mx = dtype == "mxfp4"
        self.dtype = torch.bfloat16 if self.mx else dtype
        self.chunk = int(chunk)
        self.kind = predictor.predictor

    def _weights(self):
        lins = list(self.predictor.lins)
        hid = [(_mx_weight(l) if self.mx else l.weight.detach().to(self.dtype).contiguous(),
                l.bias.detach().float().contiguous()) for l in lins[:-1]]
        head = (lins[-1].weight.detach().float().reshape(-1).contiguous(), lins[-1].bias.detach().float().contiguous())
        return hid, head

    @torch.no_grad()
    def __call__(self, h: torch.Tensor, edges: torch.Tensor) -> torch.Tensor:
        if h.device.type != "cuda":
            raise RuntimeError("EdgeScorer runs only on a HIP device (no CPU fallback)")
        h = h.to(self.dtype).contiguous()
        pairs = _as_pairs(edges.to(h.device))
        E = pairs.shape[0]
        out = torch.empty(E, dtype=torch.float32, device=h.device)
        if E == 0:
            return out
        e0 = pairs[:, 0].contiguous()
        e1 = pairs[:, 1].contiguous()
        dc = K.dtype_code(self.dtype)
        if self.kind == "inner":
            K.head_fwd(h, E, h.shape[1], None, None, prob=out, Z2=h, iz=e0, iz2=e1)
            return out
        hid, (w2, b2) = self._weights()
        for s in range(0, E, self.chunk):
            n = min(self.chunk, E - s)
            i0, i1 = e0[s:s + n], e1[s:s + n]
            if self.mx:
                z = llp_mx.quantize(h, i0, h, i1)
                for l, (W, b) in enumerate(hid):
                    z = llp_mx.linear(z, W, b, relu=True, out_dtype="mx4" if l + 1 < len(hid) else torch.bfloat16)
                K.head_fwd(z, n, z.shape[1], w2, b2, prob=out[s:s + n])
                continue
            A = K.operand(h, i0, h, i1)
            z = None
            for W, b in hid:
                z = torch.empty(n, W.shape[0], dtype=self.dtype, device=h.device)
                K.gemm_nt(A, K.operand(W), n, W.shape[0], W.shape[1], z, dc, bias=b, act=K.ACT_RELU)
                A = K.operand(z)
            K.head_fwd(z, n, z.shape[1], w2, b2, prob=out[s:s + n])
        return out


def _norm_relu(nm, h):
    """relu(norm(h)) in place, in eval mode."""
    batch = isinstance(nm, torch.nn.BatchNorm1d)
    stats = torch.empty(2, h.shape[1] if batch else h.shape[0], dtype=torch.float32, device=h.device)
    K.norm_fwd(K.NORM_BATCH if batch else K.NORM_LAYER, h, h, stats,
               None if nm.weight is None else nm.weight.detach(), None if nm.bias is None else nm.bias.detach(),
               float(nm.eps), not batch, running_mean=getattr(nm, "running_mean", None),
               running_var=getattr(nm, "running_var", None), relu=True)


def _embed_mlp_mx(layers, norms, x):
    """embed_mlp in MXFP4: hidden layers hand MXFP4 rows on (bf16 through a norm), the embedding is bf16."""
    h = x if x.dtype in (torch.float32, torch.bfloat16) else x.float()
    h = h.contiguous()
    for l, lin in enumerate(layers):
        W, b = _mx_weight(lin), lin.bias.detach().float()
        last = l == len(layers) - 1
        if norms and not last:
            h = llp_mx.linear(h, W, b, out_dtype=torch.bfloat16)
            _norm_relu(norms[l], h)
        else:
            h = llp_mx.linear(h, W, b, relu=not last, out_dtype=torch.bfloat16 if last else "mx4")
    return h


@torch.no_grad()
def embed_mlp(model, x: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """model(x) for the student MLP in eval mode (no dropout, src/models.py:45-54; with
    norm_type 'layer' / 'batch' the norm runs in eval mode, BatchNorm on its running
    statistics)."""
    if x.device.type != "cuda":
        raise RuntimeError("embed_mlp runs only on a HIP device (no CPU fallback)")
    layers = list(model.layers)
    norms = list(getattr(model, "norms", []))
    if dtype == "mxfp4":
        return _embed_mlp_mx(layers, norms, x)
    dc = K.dtype_code(dtype)
    A = K.operand(x.to(dtype).contiguous())
    h = None
    M = x.shape[0]
    for l, lin in enumerate(layers):
        last = l == len(layers) - 1
        W = lin.weight.detach().to(dtype).contiguous()
        h = torch.empty(M, W.shape[0], dtype=dtype, device=x.device)
        normed = norms and not last
        K.gemm_nt(A, K.operand(W), M, W.shape[0], W.shape[1], h, dc, bias=lin.bias.detach().float(),
                  act=K.ACT_NONE if (last or normed) else K.ACT_RELU)
        if normed:
            _norm_relu(norms[l], h)
        A = K.operand(h)
    return h


def hits_and_auc(pos: torch.Tensor, neg: torch.Tensor, Ks):
    return dict(zip(Ks, K.hits_at_k(pos, neg, Ks))), K.auc(pos, neg)


@torch.no_grad()
def test_transductive(h: torch.Tensor, predictor, split_edge, dataset: str, dtype=torch.float32):
    """src/train_teacher_gnn.py:76-155 given the node embeddings ``h``.
    Returns (results, h) with results['Hits@K'] = (valid, test), results['AUC']."""
    score = EdgeScorer(predictor, dtype)
    dev = h.device
    pv = score(h, split_edge["valid"]["edge"].to(dev))
    nv = score(h, split_edge["valid"]["edge_neg"].to(dev))
    pt = score(h, split_edge["test"]["edge"].to(dev))
    nt = score(h, split_edge["test"]["edge_neg"].to(dev))
    Ks = COLLAB_KS if dataset == "collab" else TRANSDUCTIVE_KS
    hv = K.hits_at_k(pv, nv, Ks)
    ht = K.hits_at_k(pt, nt, Ks)
    results = {f"Hits@{k}": (a, b) for k, a, b in zip(Ks, hv, ht)}
    results["AUC"] = (K.auc(pv, nv), K.auc(pt, nt))
    return results, h


@torch.no_grad()
def test_production(h_val: torch.Tensor, h_inf: torch.Tensor, predictor, val_pos, val_neg, test_edge_bundle,
                    negative_samples, dtype=torch.float32):
    """src/train_teacher_gnn.py:157-268 given the embeddings of val_data (h_val)
    and inference_data (h_inf).  test_edge_bundle = (old_old, old_new, new_new,
    test) as [2, E] tensors; negative_samples [E, 2].  Returns (results, h_val)
    with 5-tuples (val, test, old_old, old_new, new_new)."""
    score = EdgeScorer(predictor, dtype)
    dev = h_val.device
    pv = score(h_val, val_pos.to(dev))
    nv = score(h_val, val_neg.to(dev))
    oo, on, nn_, te = (t.t().to(dev) for t in test_edge_bundle)
    pt = score(h_inf, te)
    poo = score(h_inf, oo)
    pon = score(h_inf, on)
    pnn = score(h_inf, nn_)
    nt = score(h_inf, negative_samples.t().to(dev))   # negative_samples is [2, E] (src/train_teacher_gnn.py:168)
    Ks = TRANSDUCTIVE_KS
    cols = [K.hits_at_k(p, n, Ks) for p, n in ((pv, nv), (pt, nt), (poo, nt), (pon, nt), (pnn, nt))]
    results = {f"Hits@{k}": tuple(c[i] for c in cols) for i, k in enumerate(Ks)}
    results["AUC"] = tuple(K.auc(p, n) for p, n in ((pv, nv), (pt, nt), (poo, nt), (pon, nt), (pnn, nt)))
    return results, h_val
