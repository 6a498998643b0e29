"""Decoding over trees of drafted tokens (``poly_tree_chain``): what ``ChainDecoder``
does for one token of sequences of one length, for up to 64 drafted tokens of
sequences of different lengths.

A step gives every sequence a tree: node i's parent is an earlier node or (-1)
the cached tokens; -2 marks padding, so the sequences' trees may differ in
size. A node attends the cached tokens, its ancestors and itself at every level of the
chain, so its output is that of decoding its path one token at a time. The step
writes the nodes' rows behind each sequence's length; ``commit`` then keeps the
accepted path (its rows move together, the length grows) and the next step
overwrites the rest.

Lengths live on the device and every kernel reads them there, so a step or a
commit can be captured in a CUDA graph and replayed as the sequences grow. A full
cache raises ValueError in eager calls; a replay cannot, there the nodes that have
no room are padding. A decoder's steps and commits belong on one stream (or
ordered streams): its rows, lengths and workspace are one state.

16-bit caches with heads of 64 or 128 features run on the tensor cores and split a
long cache over the GPU; other types and sizes run on CUDA cores, one walk over the
cache per 8 rows.

Cache layout as ``ChainDecoder``'s (kv-head width):
  keys[t]  [b, g, cap, d]  t = 0 .. order - 1   (q2 .. q_{order + 1})
  vals[t]  [b, g, cap, d]  t = 0 .. order - 2   (v3 .. v_{order + 1})
  lses[t]  [b, g, cap]     fp32, level order - 1 first;  msgs[t] [b, g, cap, d]
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import PolyTreeAppend, PolyTreeCommit, PolyTreePass, check, lib
from .head_norm import head_rmsnorm
from .ops import _DTYPES, _no_tangents, _on, _require_cuda, _stream
from .packed import check_packed, poly_attention_chain_packed, split_heads, token_rows


def _st3(dst, t, size=1):
    s = t.stride()
    dst[0], dst[1], dst[2] = s[0] * size, s[1] * size, s[2] * size


class TreeDecoder:
    def __init__(self, *, batch, order, heads, kv_heads, dim_head, capacity, max_nodes, dtype=torch.bfloat16, device="cuda",
                 softclamp_value=None):
        if order < 2 or heads % kv_heads:
            raise ValueError("order must be at least 2 and heads divisible by kv_heads")
        if not 1 <= max_nodes <= _lib.MAX_TREE_NODES:
            raise ValueError(f"max_nodes must be in [1, {_lib.MAX_TREE_NODES}]")
        if 2 * order - 1 + 2 * (order - 1) > _lib.MAX_TREE_CACHES:
            raise ValueError("too many caches (order <= 4)")
        if dtype not in _DTYPES:
            raise TypeError(f"dtype must be one of {list(_DTYPES)}")
        if dim_head > 128:
            raise NotImplementedError("dim_head > 128 is not supported")
        self.b, self.order, self.h, self.g, self.d, self.cap = batch, order, heads, kv_heads, dim_head, capacity
        self.dtype, self.device, self.max_nodes = dtype, torch.device(device), max_nodes
        mk = lambda: torch.zeros(batch, kv_heads, capacity, dim_head, device=device, dtype=dtype)   # noqa: E731
        self.keys = [mk() for _ in range(order)]
        self.vals = [mk() for _ in range(order - 1)]
        self.msgs = [mk() for _ in range(order - 1)]
        self.lses = [torch.zeros(batch, kv_heads, capacity, device=device, dtype=torch.float32) for _ in range(order - 1)]
        self.lengths = torch.zeros(batch, device=device, dtype=torch.int32)
        self.device = self.lengths.device
        # nodes of the last step that no commit has followed; on the device, as the host does not see a replayed step
        self._step_nodes = torch.zeros(1, device=self.device, dtype=torch.int32)
        self._step_nodes_at = ctypes.c_void_p(self._step_nodes.data_ptr())
        self._bound = 0          # no sequence is longer than this ...
        self._replayed = False   # ... unless a captured commit is replayed
        self._stepped = False    # a step of the host waits for a commit
        self._captured = 0       # nodes of the largest captured step, which may have been replayed
        esz = self.keys[0].element_size()

        # one argument block per level, in launch order (element order - 1 - t is level t: queries q_{t+1}, keys q_{t+2})
        self._passes = (PolyTreePass * order)()
        for t in range(order - 1, -1, -1):
            a = self._passes[order - 1 - t]
            a.batch, a.heads, a.kv_heads, a.head_dim = batch, heads if t == 0 else kv_heads, kv_heads, dim_head
            a.dtype, a.capacity, a.scale = _DTYPES[dtype], capacity, dim_head ** -0.5
            a.softclamp = float(softclamp_value) if softclamp_value else 0.0
            a.k = self.keys[t].data_ptr()
            _st3(a.k_stride, self.keys[t])
            val = self.vals[-1] if t == order - 1 else self.vals[t - 1] if t else self.msgs[order - 2]
            a.v = val.data_ptr()
            _st3(a.v_stride, val)
            if 0 < t < order - 1:
                mul = self.msgs[order - 2 - t]
                a.v_mul = mul.data_ptr()
                _st3(a.v_mul_stride, mul)
            if t < order - 1:
                bias = self.lses[order - 2 - t]
                a.bias = bias.data_ptr()
                a.bias_stride[0], a.bias_stride[1] = bias.stride(0), bias.stride(1)
            if t >= 1:
                msg, lse = self.msgs[order - 1 - t], self.lses[order - 1 - t]
                a.cache_out, a.cache_lse = msg.data_ptr(), lse.data_ptr()
                _st3(a.cache_out_stride, msg)
                a.cache_lse_stride[0], a.cache_lse_stride[1] = lse.stride(0), lse.stride(1)
            a.lengths = self.lengths.data_ptr()
        # the rows a step appends, and all the rows a commit moves
        self._append = PolyTreeAppend()
        self._append.batch, self._append.kv_heads, self._append.row_bytes = batch, kv_heads, dim_head * esz
        self._append.capacity, self._append.lengths = capacity, self.lengths.data_ptr()
        self._append.n = 2 * order - 1
        for r, c in zip(self._append.t, self.keys + self.vals):
            r.cache = c.data_ptr()
            _st3(r.cache_stride, c, esz)
        self._commit = PolyTreeCommit()
        self._commit.batch, self._commit.kv_heads, self._commit.capacity = batch, kv_heads, capacity
        self._commit.lengths = self.lengths.data_ptr()
        caches = self.keys + self.vals + self.msgs + [x.unsqueeze(-1) for x in self.lses]
        self._commit.n = len(caches)
        for r, c in zip(self._commit.t, caches):
            r.cache, r.row_bytes = c.data_ptr(), c.shape[-1] * c.element_size()
            _st3(r.cache_stride, c, c.element_size())
        # one workspace that every step fits in (the passes of a step use it one after another)
        need = 0
        for a in self._passes:
            a.q = a.parents = a.k      # any address: only the sizes count
            with _on(self.device):
                for n in range(1, max_nodes + 1):
                    a.nodes = n
                    need = max(need, lib.poly_tree_workspace_size(a))
        self._ws = torch.empty(max(need, 1), device=device, dtype=torch.uint8)
        for a in self._passes:
            a.workspace, a.workspace_bytes = self._ws.data_ptr(), need

    # ------------------------------------------------------------------ contents
    def load(self, keys, vals, lses, msgs, lengths):
        """Cached rows of every sequence: keys / vals / msgs [b, g, n, d] and lses [b, g, n] of n <= capacity rows,
        of which sequence i uses the first lengths[i] (a list or an integer tensor [b])."""
        lengths = torch.as_tensor(lengths)
        if lengths.numel() and (lengths.is_floating_point() or lengths.is_complex() or lengths.dtype == torch.bool):
            raise TypeError(f"lengths must be integers, got {lengths.dtype}")
        longest = int(lengths.max()) if lengths.numel() else 0
        if lengths.shape != (self.b,) or (lengths.numel() and int(lengths.min()) < 0):
            raise ValueError(f"lengths must be [{self.b}] and non-negative")
        if any(len(x) != n for x, n in ((keys, self.order), (vals, self.order - 1), (lses, self.order - 1), (msgs, self.order - 1))):
            raise ValueError("an order-n decoder holds n key caches and n - 1 of values, lses and messages")
        pairs = list(zip(self.keys + self.vals + self.msgs + self.lses, (*keys, *vals, *msgs, *lses)))
        for c, t in pairs:      # all of them before the first is written
            if (t.dim() != c.dim() or longest > t.shape[2] or t.shape[2] > self.cap or t.shape[:2] != c.shape[:2]
                    or t.shape[3:] != c.shape[3:]):
                raise ValueError(f"cache rows {tuple(t.shape)} do not fit {tuple(c.shape)} and lengths up to {longest}")
        for c, t in pairs:
            c[:, :, :t.shape[2]].copy_(t.detach())
        self.lengths.copy_(lengths)
        self._step_nodes.zero_()
        self._bound, self._stepped = longest, False

    def load_packed(self, keys, vals, lses, msgs, cu_seqlens, max_seqlen):
        """The same from a packed prompt batch: keys / vals / msgs [total, g, d], lses [g, total] (what
        ``poly_attention_chain_packed`` takes and returns), sequence i being rows cu_seqlens[i] .. cu_seqlens[i + 1].
        ``max_seqlen`` bounds the lengths; the sequences themselves have to fit the capacity."""
        if cu_seqlens.shape[0] != self.b + 1:
            raise ValueError(f"cu_seqlens must hold {self.b} sequences")
        start = cu_seqlens[:-1].long()
        rows = start[:, None] + torch.arange(min(max_seqlen, self.cap), device=start.device)
        rows = rows.clamp_(0, max(keys[0].shape[0] - 1, 0))
        pick = lambda t: t[rows].permute(0, 2, 1, 3)   # noqa: E731
        self.load([pick(t) for t in keys], [pick(t) for t in vals], [t.t()[rows].permute(0, 2, 1) for t in lses],
                  [pick(t) for t in msgs], (cu_seqlens[1:] - cu_seqlens[:-1]))

    def refresh(self):
        """Waits for the device and tightens the host's bound of the lengths; returns it."""
        self._bound = int(self.lengths.max()) if self.b else 0
        return self._bound

    def _room(self, nodes):
        if self._replayed or self._bound + nodes > self.cap:
            if not torch.cuda.is_current_stream_capturing() and self.refresh() + nodes > self.cap:
                raise ValueError("KV cache capacity exceeded")

    def _parents(self, parents, nodes):
        _require_cuda(parents)
        if parents.dtype != torch.int32 or parents.device != self.device:
            raise TypeError("parents must be an int32 tensor on the decoder's device")
        if parents.dim() == 1:
            parents = parents.unsqueeze(0).expand(self.b, -1)
        if parents.shape != (self.b, nodes):
            raise ValueError(f"parents must be [{self.b}, {nodes}] or [{nodes}], got {tuple(parents.shape)}")
        return parents if parents.stride(1) == 1 or nodes == 1 else parents.contiguous()

    # ------------------------------------------------------------------ steps
    def positions(self, parents):
        """Every node's position in its sequence, int32 [b, nodes] (length plus depth), e.g. for its rotary angles."""
        nodes = parents.shape[-1]
        parents = self._parents(parents, nodes)
        out = torch.empty(self.b, nodes, device=self.device, dtype=torch.int32)
        with _on(self.device):
            check(lib.poly_tree_positions(self.lengths.data_ptr(), parents.data_ptr(), parents.stride(0), self.b, nodes,
                                          out.data_ptr(), out.stride(0), _stream(self.device)), "poly_tree_positions")
        return out

    def step(self, q1, new_keys, new_vals, parents, *, out=None, return_rows=False):
        """Append the nodes' rows and run the chain for them.

        q1 [b, h, T, d]; new_keys (order) and new_vals (order - 1) [b, g, T, d]; parents int32 [b, T] (or [T] for
        all). Returns out [b, h, T, d], or with ``return_rows`` (out, msgs, lses): the nodes' messages [b, g, T, d] and
        log-sum-exps [b, g, T] of every level, in the caches' order. Padding nodes come out as zeros. Results carry no
        gradients, whether or not the inputs require them.
        """
        b, order, g = self.b, self.order, self.g
        news = [*new_keys, *new_vals]
        nodes = q1.shape[2] if q1.dim() == 4 else -1
        if q1.shape != (b, self.h, nodes, self.d) or not 1 <= nodes <= self.max_nodes:
            raise ValueError(f"q1 must be [{b}, {self.h}, 1..{self.max_nodes}, {self.d}], got {tuple(q1.shape)}")
        if len(new_keys) != order or len(new_vals) != order - 1 or any(t.shape != (b, g, nodes, self.d) for t in news):
            raise ValueError(f"a step takes {order} key and {order - 1} value tensors [{b}, {g}, {nodes}, {self.d}]")
        for t in (q1, *news):
            if not t.is_cuda:
                _require_cuda(t)
            if t.dtype != self.dtype or t.device != self.device:
                raise TypeError(f"tree tensors must be {self.dtype} on {self.device}")
        _no_tangents(news, q1)
        parents = self._parents(parents, nodes)
        self._room(nodes)
        rows = lambda t: t if t.stride(-1) == 1 else t.contiguous()   # noqa: E731
        q1, news = rows(q1), [rows(t) for t in news]
        if out is None:
            out = torch.empty(b, self.h, nodes, self.d, device=self.device, dtype=self.dtype)
        elif out.shape != q1.shape or out.dtype != self.dtype or out.device != self.device or out.stride(-1) != 1:
            raise ValueError("out must have q1's shape, dtype and device and a contiguous last dim")
        ap, esz = self._append, q1.element_size()
        ap.nodes, ap.parents, ap.parents_stride = nodes, parents.data_ptr(), parents.stride(0)
        for r, t in zip(ap.t, news):
            r.src = t.data_ptr()
            _st3(r.src_stride, t, esz)
        msgs, lses = [], []
        if b == 0:      # no sequence: nothing to append (empty tensors have no address for the library)
            if return_rows:
                msgs = [torch.empty(0, g, nodes, self.d, device=self.device, dtype=self.dtype) for _ in range(order - 1)]
                lses = [torch.empty(0, g, nodes, device=self.device, dtype=torch.float32) for _ in range(order - 1)]
            self._stepped = True
            return (out, msgs, lses) if return_rows else out
        for t in range(order - 1, -1, -1):
            a = self._passes[order - 1 - t]
            q = q1 if t == 0 else news[t - 1]
            a.nodes, a.parents, a.parents_stride = nodes, ap.parents, ap.parents_stride
            a.q = q.data_ptr()
            _st3(a.q_stride, q)
            if t == 0:
                a.out = out.data_ptr()
                _st3(a.out_stride, out)
            elif return_rows:
                m = torch.empty(b, g, nodes, self.d, device=self.device, dtype=self.dtype)
                s = torch.empty(b, g, nodes, device=self.device, dtype=torch.float32)
                a.out, a.lse = m.data_ptr(), s.data_ptr()
                _st3(a.out_stride, m)
                a.lse_stride[0], a.lse_stride[1] = s.stride(0), s.stride(1)
                msgs.append(m)
                lses.append(s)
            else:
                a.out = a.lse = None
        with _on(self.device):
            check(lib.poly_tree_chain_counted(ap, self._passes, order, self._step_nodes_at, _stream(self.device)), "poly_tree_chain")
        self._stepped = True
        if torch.cuda.is_current_stream_capturing():
            self._captured = max(self._captured, nodes)
        return (out, msgs, lses) if return_rows else out

    def commit(self, path, count):
        """Keep, of the last step's nodes, path[i, :count[i]] (int32 [b, n], ascending node indices) of each sequence;
        count int32 [b]. Both stay on the device. An entry past those nodes is their last one, a count is at most their
        number, and a second commit keeps nothing (it raises, unless a captured step may have been replayed since)."""
        _require_cuda(path, count)
        if path.dtype != torch.int32 or count.dtype != torch.int32 or path.device != self.device or count.device != self.device:
            raise TypeError("path and count must be int32 tensors on the decoder's device")
        if path.dim() != 2 or path.shape[0] != self.b or path.shape[1] < 1 or count.shape != (self.b,):
            raise ValueError(f"path must be [{self.b}, n] and count [{self.b}]")
        if not (self._stepped or self._captured):
            raise ValueError("nothing to commit: no step since the last commit")
        path, count = path if path.stride(1) == 1 else path.contiguous(), count.contiguous()
        c = self._commit
        c.nodes, c.path_len = max(self._append.nodes, self._captured), path.shape[1]   # at most; _step_nodes says which
        c.path, c.path_stride, c.count = path.data_ptr(), path.stride(0), count.data_ptr()
        if self.b == 0:
            self._stepped = False
            return
        with _on(self.device):
            check(lib.poly_tree_commit_counted(c, self._step_nodes_at, _stream(self.device)), "poly_tree_commit")
        self._stepped = False
        self._replayed = self._replayed or torch.cuda.is_current_stream_capturing()
        self._bound = min(self.cap, self._bound + min(c.nodes, c.path_len))


class TreeDecoding:
    """Drafted-token decoding of the attention modules (``PolyAttention``, ``NPolyAttention``; causal ones): a packed
    prompt batch fills a ``TreeDecoder``, then each step runs a tree of tokens per sequence through the module. With
    ``use_rotary_embed`` the decoder holds rotated keys, every token at its position in its sequence."""

    def _tree_project(self, x):
        order = len(self.to_kvs)
        normed = self.norm(x)
        contexts = [norm(x) for norm in self.context_norms] if self.context_norms is not None else [normed] * order
        qg = split_heads(self.to_q(normed), self.q_split, self.heads)
        kvs = [split_heads(to_kv(c), self.kv1_split if i == 0 else self.kv_split, self.kv_heads)
               for i, (to_kv, c) in enumerate(zip(self.to_kvs, contexts))]
        if self.shared_kv:
            root, vs = kvs[0][0], [kv[0] for kv in kvs[1:]]
        else:
            root, vs = kvs[0][1] if self.has_root_v else None, [kv[1] for kv in kvs[1:]]
        qs = head_rmsnorm(self.q_norms, (qg[0], *(kv[0] for kv in kvs)))
        return list(qs), vs, root, qg[1] if self.attn_gate else None

    @torch.no_grad()
    def tree_prefill(self, x, cu_seqlens, *, max_seqlen, capacity, max_nodes):
        """Prompts x [1, total, dim] packed by cu_seqlens -> (y [1, total, dim], TreeDecoder of the sequences)."""
        if not self.causal:
            raise ValueError("decoding needs a causal module")
        check_packed(x)
        qs, vs, root, gates = self._tree_project(x)
        if self.rotary_emb is not None:
            qs = self.rotary_emb(qs, cu_seqlens=cu_seqlens)
        qs, vals = [token_rows(q) for q in qs], [token_rows(v) for v in vs]
        out, lses, msgs = poly_attention_chain_packed([qs[0], *qs[1:-1]], qs[1:], vals, cu_seqlens,
                                                      softclamp_value=self.softclamp_value, causal=True, max_seqlen=max_seqlen)
        dec = TreeDecoder(batch=cu_seqlens.shape[0] - 1, order=len(vs) + 1, heads=self.heads, kv_heads=self.kv_heads,
                          dim_head=self.dim_head, capacity=capacity, max_nodes=max_nodes, dtype=out.dtype, device=out.device,
                          softclamp_value=self.softclamp_value)
        dec.load_packed(qs[1:], vals, lses, msgs, cu_seqlens, max_seqlen)
        return self._finish(out.transpose(0, 1).unsqueeze(0), root, gates), dec

    @torch.no_grad()
    def tree_step(self, x, decoder, parents):
        """Drafted tokens x [b, T, dim] with their trees (``TreeDecoder.step``) -> y [b, T, dim]. ``decoder.commit`` then
        keeps the accepted ones."""
        qs, vs, root, gates = self._tree_project(x)
        if self.rotary_emb is not None:
            qs = self.rotary_emb(qs, positions=decoder.positions(parents))
        return self._finish(decoder.step(qs[0], qs[1:], vs, parents), root, gates)


__all__ = ["TreeDecoder", "TreeDecoding"]
