"""The encoders of the reference with its class names, constructor arguments and state_dict keys (models.py:8-80 GraphConv,
:83-316 GcnEncoderGraph, :330-380 GcnEncoderNode), so that `explainer_main.py` can rebuild an encoder and `load_state_dict` a
reference checkpoint without importing the reference.

The HIP engine reads only the frozen weights of the default configuration (3 layers, bias, method "base": `model.state_dict()`).
`forward` is a plain torch restatement of the reference's forward: predictions outside the hot path, and the model the torch
route of the explainer (explainer/torch_route.py) differentiates through for the configurations the kernels do not implement -
`method="att"` (models.py:62-68: adj * (x W_att)(x W_att)^T per layer), any number of layers, `add_self`, dropout.

Two options the reference does not have, both read from `args`, both on the kernels of ops.py where the model is on the GPU:
  layer_norm    True: a learned LayerNorm after the ReLU of every hidden layer in the place of apply_bn (state_dict keys norms.<layer>.weight / .bias);
  dropout_seed  an int: the layers' dropout draws its masks from (seed, use, layer, node, feature) instead of torch's generator, so that a training run or an
                explanation through the torch route is reproducible by itself; `reset_dropout()` starts the uses again, `forward(..., dropout_use=n)` draws the
                n-th use's whatever ran before (what a forward pass that is run again, as by torch.utils.checkpoint, needs).
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops


class LayerNorm(nn.Module):
    """LayerNorm over the features of relu(x), one gain and offset per feature; on the GPU one kernel (ops.layer_norm), the ReLU in it, for x in float32, bfloat16 or
    float16 (other types are refused there)."""

    def __init__(self, dim, eps=1e-5):
        super().__init__()
        self.dim, self.eps = dim, eps
        self.weight = nn.Parameter(torch.ones(dim))
        self.bias = nn.Parameter(torch.zeros(dim))

    def forward(self, x):
        if x.is_cuda or ops._ENGINE["lib"] is not None:
            return ops.layer_norm(x, self.weight, self.bias, self.eps, relu=True)
        return F.layer_norm(F.relu(x), (self.dim,), self.weight, self.bias, self.eps)

    def with_dropout(self, x, drop, use=None, row_offset=0):
        """(self(x), drop(self(x), use, row_offset)) in one pass each way (ops.layer_norm_dropout)."""
        return ops.layer_norm_dropout(x, self.weight, self.bias, drop.p, drop.seed, drop.step(use), self.eps, relu=True, row_offset=row_offset)


class CounterDropout(nn.Module):
    """Dropout whose mask is a function of (seed, use, layer, row, feature): ops.dropout.  `use` is the caller's number of this forward pass; left out, `uses` counts the
    calls in training mode on the host and is part of the state_dict: a training run that is resumed goes on with the masks that come next.  A forward pass that is run
    again must draw the masks it drew first, which a count of calls cannot know: inside a backward pass (recomputation, torch.utils.checkpoint) the use has to be given.
    row_offset: where x's rows begin in the whole of which they are a shard.  A step captured into a graph repeats the use it was captured with (ops.dropout takes a
    seed tensor for new masks at every replay)."""

    def __init__(self, p, seed, layer, layers):
        super().__init__()
        self.p, self.seed, self.layer, self.layers, self.uses = float(p), int(seed), layer, layers, 0

    def step(self, use=None):
        """The generator's step of the given use, or of the next one."""
        if getattr(self, "_is_replica", False):
            raise RuntimeError("seeded dropout in a replica of torch.nn.DataParallel: every replica would draw the same masks, and their count of uses is thrown away "
                               "with them; run one process per GPU, each with its first_graph=")
        if use is None:
            if torch._C._current_graph_task_id() != -1:
                raise RuntimeError("dropout drawn by a count of its calls, inside a backward pass: a recomputed forward pass would draw other masks than the first one; "
                                   "pass the number of the training step, dropout_use= to the encoder (use= to CounterDropout), in both")
            use = self.uses
            self.uses += 1
        return use * self.layers + self.layer

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        destination[prefix + "uses"] = torch.tensor(self.uses)

    def _load_from_state_dict(self, state_dict, prefix, *rest):
        uses = state_dict.pop(prefix + "uses", None)      # (a state_dict from an encoder without such dropout has none: the count stays)
        if uses is not None:
            self.uses = int(uses)
        super()._load_from_state_dict(state_dict, prefix, *rest)

    def forward(self, x, use=None, row_offset=0):
        return ops.dropout(x, self.p, self.seed, self.step(use), row_offset) if self.training else x


class GraphConv(nn.Module):
    """y = normalize((adj' x) W (+ x W_self) + b), adj' = adj * att with att = (x W_att)(x W_att)^T when `att` (models.py:58-80)."""

    def __init__(self, input_dim, output_dim, add_self=False, normalize_embedding=False, dropout=0.0, bias=True, gpu=True, att=False,
                 dropout_layer=None):
        super().__init__()
        self.att, self.add_self, self.dropout, self.normalize_embedding = att, add_self, dropout, normalize_embedding
        self.input_dim, self.output_dim = input_dim, output_dim
        if dropout > 0.001:
            self.dropout_layer = nn.Dropout(p=dropout) if dropout_layer is None else dropout_layer
        self.weight = nn.Parameter(torch.empty(input_dim, output_dim))
        if add_self:
            self.self_weight = nn.Parameter(torch.empty(input_dim, output_dim))
        if att:
            self.att_weight = nn.Parameter(torch.empty(input_dim, input_dim))
        self.bias = nn.Parameter(torch.zeros(output_dim)) if bias else None

    def counter_dropout(self):
        """The layer's CounterDropout where it is to be applied now, else None."""
        drop = self.dropout_layer if self.dropout > 0.001 else None
        return drop if isinstance(drop, CounterDropout) and drop.training else None

    def _load_from_state_dict(self, state_dict, prefix, *rest):
        if not isinstance(getattr(self, "dropout_layer", None), CounterDropout):
            state_dict.pop(prefix + "dropout_layer.uses", None)      # the count of another encoder's CounterDropout
        super()._load_from_state_dict(state_dict, prefix, *rest)

    def forward(self, x, adj, dropped=False):
        """dropped: x has been through this layer's dropout already (LayerNorm.with_dropout)."""
        if self.dropout > 0.001 and not dropped:
            x = self.dropout_layer(x)
        if self.att:
            x_att = torch.matmul(x, self.att_weight)
            adj = adj * (x_att @ x_att.permute(0, 2, 1))
        y = torch.matmul(torch.matmul(adj, x), self.weight)
        if self.add_self:
            y = y + torch.matmul(x, self.self_weight)
        if self.bias is not None:
            y = y + self.bias
        if self.normalize_embedding:
            y = F.normalize(y, p=2, dim=2)
        return y, adj


class GcnEncoderGraph(nn.Module):
    def __init__(self, input_dim, hidden_dim, embedding_dim, label_dim, num_layers, pred_hidden_dims=(), concat=True,
                 bn=True, dropout=0.0, add_self=False, args=None):
        super().__init__()
        self.concat, self.bn, self.num_layers, self.num_aggs = concat, bool(bn), num_layers, 1
        self.bias = True if args is None else getattr(args, "bias", True)
        self.att = args is not None and getattr(args, "method", "base") == "att"
        seed = None if args is None else getattr(args, "dropout_seed", None)
        counter = lambda layer: None if seed is None or not dropout > 0.001 else CounterDropout(dropout, seed, layer, num_layers - 2)
        gc = lambda i, o, dp=0.0, drop=None: GraphConv(i, o, add_self=add_self, normalize_embedding=True, dropout=dp, bias=self.bias, att=self.att,
                                                       dropout_layer=drop)
        self.conv_first = gc(input_dim, hidden_dim)
        self.conv_block = nn.ModuleList([gc(hidden_dim, hidden_dim, dropout, counter(i)) for i in range(num_layers - 2)])
        self.conv_last = gc(hidden_dim, embedding_dim)
        self.norms = None
        if args is not None and getattr(args, "layer_norm", False):
            if self.bn:
                raise ValueError("bn and layer_norm are two normalisations of the same rows: choose one")
            self.norms = nn.ModuleList([LayerNorm(hidden_dim) for _ in range(len(self.conv_block) + 1)])
        self.act = nn.ReLU()
        self.label_dim = label_dim
        self.pred_input_dim = hidden_dim * (num_layers - 1) + embedding_dim if concat else embedding_dim
        if len(pred_hidden_dims) == 0:
            self.pred_model = nn.Linear(self.pred_input_dim, label_dim)
        else:
            layers, d = [], self.pred_input_dim
            for h in pred_hidden_dims:
                layers += [nn.Linear(d, h), self.act]
                d = h
            layers.append(nn.Linear(d, label_dim))
            self.pred_model = nn.Sequential(*layers)
        gain = nn.init.calculate_gain("relu")
        for m in self.modules():
            if isinstance(m, GraphConv):
                nn.init.xavier_uniform_(m.weight.data, gain=gain)
                if m.att:
                    nn.init.xavier_uniform_(m.att_weight.data, gain=gain)
                if m.add_self:
                    nn.init.xavier_uniform_(m.self_weight.data, gain=gain)

    def apply_bn(self, x):
        """models.py:222-228: a fresh BatchNorm1d(num_nodes) in training mode - every node standardised over its features."""
        return F.batch_norm(x, None, None, None, None, True, 0.1, 1e-5)

    def reset_dropout(self, uses=None):
        """Every CounterDropout starts its uses again: what follows draws the masks that a new model would.  Returns the counts so far, with which (as `uses`) another
        call goes on where they were."""
        drops = [m for m in self.modules() if isinstance(m, CounterDropout)]
        before = [m.uses for m in drops]
        for m, n in zip(drops, uses or [0] * len(drops)):
            m.uses = n
        return before

    def _activate(self, layer, x, nxt, use, row_offset):
        """What follows graph convolution `layer` (models.py:239-253): (the layer's embedding, what convolution `nxt` reads, whether that has been through its
        dropout)."""
        drop = nxt.counter_dropout()
        if self.norms is not None:
            if drop is not None:
                h, d = self.norms[layer].with_dropout(x, drop, use, row_offset)
                return h, d, True
            x = self.norms[layer](x)
            return x, x, False
        x = self.act(x)
        if self.bn:
            x = self.apply_bn(x)
        if drop is not None:
            return x, drop(x, use, row_offset), True
        return x, x, False

    def _layers(self, x, adj, dropout_use=None, first_graph=0):
        """The graph convolutions one after the other: (embedding, attention adjacency) of each."""
        convs = [self.conv_first, *self.conv_block, self.conv_last]
        dropped = False
        for i, conv in enumerate(convs):
            x, adj_att = conv(x, adj, dropped)
            if i + 1 == len(convs):
                yield x, adj_att
                return
            h, x, dropped = self._activate(i, x, convs[i + 1], dropout_use, first_graph * adj.shape[-1])
            yield h, adj_att

    def gcn_forward(self, x, adj, dropout_use=None, first_graph=0):
        """models.py:230-267: all layers, concatenated embeddings [1, n, H (L - 1) + O] and the stacked attention adjacencies (the
        block layers re-append conv_first's, as the reference does at :252)."""
        x_all, att_all = [], []
        for i, (h, adj_att) in enumerate(self._layers(x, adj, dropout_use, first_graph)):
            x_all.append(h)
            att_all.append(att_all[0] if 0 < i <= len(self.conv_block) else adj_att)
        return torch.cat(x_all, dim=2), torch.stack(att_all, dim=3)

    def forward(self, x, adj, batch_num_nodes=None, dropout_use=None, first_graph=0, **kwargs):
        """models.py:269-316: per-layer max over all rows, concat, linear head.  dropout_use: CounterDropout's use;
        first_graph: the first graph's number in the whole batch of which this is a rank's share (its rows are counted from there)."""
        outs, atts = [], []
        for h, adj_att in self._layers(x, adj, dropout_use, first_graph):
            outs.append(h.max(dim=1)[0])
            atts.append(adj_att)
        output = torch.cat(outs, dim=1) if self.concat else outs[-1]
        return self.pred_model(output), torch.stack(atts, dim=3)


class GcnEncoderNode(GcnEncoderGraph):
    def forward(self, x, adj, batch_num_nodes=None, dropout_use=None, first_graph=0, **kwargs):
        """models.py:363-376: the head on every row.  dropout_use: CounterDropout's use;
        first_graph: the first graph's number in the whole batch of which this is a rank's share (its rows are counted from there)."""
        emb, adj_att = self.gcn_forward(x, adj, dropout_use, first_graph)
        return self.pred_model(emb), adj_att
