"""Host mirror of network/experiment.py (Experiment :23-224) and of the classifier trainer on config 4's path
(finetuner.CIFAR10.pass_samples :199-246, ethec_experiments.ETHECExperiment :202-240): model forward -> criterion ->
backward -> optimizer step, with the CNN parameters in one flat arena (single all-reduce, single Adam launch)."""
import copy
import os
import time

import torch
import torch.nn as nn

from . import parallel
from .loss import path_log_probs
from .quant import MXFP4Linear
from .resnet import resnet18, resnet50


class _NullWriter:
    def add_scalar(self, *a, **k): pass
    def close(self): pass


class Experiment:
    """experiment.py:23-224: epoch loop, MultiStepLR, checkpoints.  `evaluator` may be None (host-side reporting is
    out of scope); `pass_samples` is the base (inputs, labels) variant."""

    def __init__(self, model, dataloaders, criterion, classes, experiment_name, n_epochs, eval_interval, batch_size,
                 exp_dir, load_wt, evaluator, lr_step=[]):
        self.epoch = 0
        self.exp_dir = exp_dir; self.load_wt = load_wt; self.eval = evaluator
        self.classes = classes; self.criterion = criterion; self.batch_size = batch_size
        if not torch.cuda.is_available():
            raise RuntimeError('Experiment runs on the MI355X only (no CPU fallback)')
        self.device = torch.device('cuda', torch.cuda.current_device())
        print('Using device: {}'.format(self.device))
        self.model = model.to(self.device)
        self.n_epochs = n_epochs; self.eval_interval = eval_interval; self.dataloaders = dataloaders
        self.log_dir = os.path.join(self.exp_dir, '{}').format(experiment_name)
        self.path_to_save_model = os.path.join(self.log_dir, 'weights')
        self.make_dir_if_non_existent(self.path_to_save_model)
        self.writer = _NullWriter()
        self.lr_step = lr_step
        self.best_score = 0.0; self.best_model_wts = None

    @staticmethod
    def make_dir_if_non_existent(dir):
        if not os.path.exists(dir):
            os.makedirs(dir, exist_ok=True)

    def set_parameter_requires_grad(self, feature_extracting):
        if feature_extracting:
            for param in self.model.parameters():
                param.requires_grad = False

    def pass_samples(self, phase, save_to_tensorboard=True):
        running_loss = torch.zeros((), device=self.device); n = 0
        self.model.train(phase == 'train')
        for inputs, labels in self.dataloaders[phase]:
            inputs = inputs.to(self.device); labels = labels.to(self.device)
            self.optimizer.zero_grad()
            with torch.set_grad_enabled(phase == 'train'):
                outputs = self.model(inputs)
                loss = self.criterion(outputs, labels)
                if phase == 'train':
                    loss.backward(); self.optimizer.step()
            running_loss += loss.detach() * inputs.size(0); n += inputs.size(0)
        epoch_loss = running_loss.item() / max(n, 1)
        print('{} Loss: {:.4f}'.format(phase, epoch_loss))
        return epoch_loss

    def run_model(self, optimizer):
        self.optimizer = optimizer
        scheduler = torch.optim.lr_scheduler.MultiStepLR(self.optimizer, milestones=self.lr_step, gamma=0.1)
        if self.load_wt:
            self.find_existing_weights()
        self.best_model_wts = copy.deepcopy(self.model.state_dict()); self.best_score = 0.0
        since = time.time()
        for self.epoch in range(self.epoch, self.n_epochs):
            print('=' * 10); print('Epoch {}/{}'.format(self.epoch, self.n_epochs - 1)); print('=' * 10)
            self.pass_samples(phase='train')
            if self.epoch % self.eval_interval == 0:
                self.pass_samples(phase='val'); self.pass_samples(phase='test')
            scheduler.step()
        print('Training complete in {:.0f}s'.format(time.time() - since))
        self.writer.close()
        return self.model

    def save_model(self, loss, filename=None):
        torch.save({'epoch': self.epoch, 'model_state_dict': self.model.state_dict(),
                    'optimizer_state_dict': self.optimizer.state_dict(), 'loss': loss},
                   os.path.join(self.path_to_save_model, '{}.pth'.format(filename if filename else self.epoch)))

    def load_model(self, epoch_to_load):
        ck = torch.load(os.path.join(self.path_to_save_model, '{}.pth'.format(epoch_to_load)), map_location=self.device)
        self.model.load_state_dict(ck['model_state_dict']); self.model = self.model.to(self.device)
        self.optimizer.load_state_dict(ck['optimizer_state_dict']); self.epoch = ck['epoch']

    def find_existing_weights(self):
        weights = sorted(os.listdir(self.path_to_save_model))
        if len(weights) < 2:
            print('Could not find weights to load from, will train from scratch.')
        else:
            self.load_model(epoch_to_load=weights[-2].split('.')[0])


class ETHECExperiment(Experiment):
    """Config 4's trainer: finetuner.CIFAR10 (model zoo pick :121-122, fc swap :150-157, pass_samples :199-246) as used
    by ethec_experiments.ETHECExperiment (:202-240).  criterion(outputs, labels, level_labels) -> scalar."""

    def __init__(self, data_loaders, labelmap, criterion, lr, batch_size=8, evaluator=None, experiment_name='exp',
                 experiment_dir='../exp/', n_epochs=10, eval_interval=2, feature_extracting=False, use_pretrained=False,
                 load_wt=False, model_name='resnet50', optimizer_method='adam', compute_dtype=torch.float32, weights=None, fast_path=True):
        self.labelmap = labelmap; self.lr = lr; self.model_name = model_name
        self.n_classes = labelmap.n_classes; self.levels = labelmap.levels; self.n_levels = len(labelmap.levels)
        self.rank, self.local_rank, self.world = parallel.init_process_group()
        if self.world > 1:
            torch.cuda.set_device(self.local_rank % torch.cuda.device_count())
        model = {'resnet18': resnet18, 'resnet50': resnet50}[model_name]()
        if weights is not None:
            model.load_state_dict(weights)
        model.fc = nn.Linear(model.fc.in_features, self.n_classes)          # finetuner.py:150-157
        model = model.to(memory_format=torch.channels_last)
        Experiment.__init__(self, model, data_loaders, criterion, labelmap.classes, experiment_name, n_epochs,
                            eval_interval, batch_size, experiment_dir, load_wt, evaluator)
        self.compute_dtype = compute_dtype
        self.arena = parallel.FlatArena(self.model.parameters(), self.device)
        self.reducer = parallel.GradientReducer(self.arena)
        if self.world > 1:
            torch.distributed.broadcast(self.arena.data, 0)
        # liblecone's convolutions / fused BatchNorm / arena gradients / side-stream weight gradients, as in engine.StepEngine
        from .resnet import WgradOverlap
        self.overlap = None
        if fast_path and compute_dtype in (torch.float32, torch.bfloat16):
            if compute_dtype == torch.bfloat16:
                self.arena.enable_lowp_transposed()     # bf16 shadow + its transposed twin (the data gradients' operand)
            self.overlap = WgradOverlap(self.reducer, self.arena, side_stream=True)
        self.model.wgrad_overlap = self.overlap if self.overlap is not None else False    # this trainer's own (resnet.ResNet.wgrad_overlap)

    def fwd_bwd(self, inputs, level_labels, labels=None):
        """Forward, criterion, backward of one batch already on the device (NHWC): the region a hipGraph can capture."""
        self.arena.zero_grad()
        with torch.autocast('cuda', dtype=self.compute_dtype, enabled=self.compute_dtype != torch.float32):
            outputs = self.model(inputs)
        loss = self.criterion(outputs.float(), labels, level_labels)
        loss.backward()
        if self.overlap is not None:
            self.overlap.join()
        # detached: a live `outputs` would keep this step's autograd graph (and its AccumulateGrad nodes, bound to this step's
        # stream) alive into the next one -- under hipGraph capture that ends in a crash inside capture_end
        return loss.detach(), outputs.detach()

    def train_step(self, inputs, labels, level_labels):
        """finetuner.py:213-246 for one batch: forward, criterion, backward, (SUM all-reduce), Adam.  The criterion's
        mean is over the LOCAL batch, so under DP the summed gradient is divided by the world size."""
        pend = self.__dict__.setdefault('_steps_in_flight', [])     # host at most two steps ahead (see JointEmbeddings.train_step)
        if len(pend) >= 2:
            pend.pop(0).synchronize()
        inputs = inputs.to(self.device, non_blocking=True).contiguous(memory_format=torch.channels_last)
        loss, outputs = self.fwd_bwd(inputs, level_labels.to(self.device), labels)
        self.reducer.finish()
        self.arena.adam_step(self.lr, grad_scale=1.0 / self.world)
        if loss.is_cuda:
            done = torch.cuda.Event(); done.record(); pend.append(done)
        return loss, outputs

    # ---- learning from feedback on the model's answers (label paths) instead of labels; no counterpart in the reference
    def freeze_reference(self, head='mxfp4'):
        """Keeps a frozen copy of the present model as `self.reference` -- what the preference loss and the KL term measure against.  head: 'mxfp4' holds the classifier
        in 4 bits (a quarter of bf16's weights; its log-probabilities are close to, not equal to, the model's; faster than bf16 from heads of 10 000 x 2 048 on, smaller ones from
        512 to 4 096 rows -- for 723 classes it saves no time beyond a single row), 'full' keeps it as it is.  The copy is in
        no checkpoint: to go on with a run, load the model it was taken from, call this, then load the run's."""
        if head not in ('mxfp4', 'full'):
            raise ValueError("head must be 'mxfp4' or 'full', got %r" % (head,))
        ref = copy.deepcopy(self.model)
        for p in ref.parameters():
            p.requires_grad = False
        ref.wgrad_overlap = False
        if head == 'mxfp4':
            ref.fc = MXFP4Linear.from_linear(ref.fc, out_dtype=torch.float32)
        self.reference = ref.eval()
        return self.reference

    def reference_log_probs(self, inputs, paths):
        """Log-probabilities of paths ([B, L] or [B, G, L], see loss.path_log_probs) under the frozen reference."""
        if getattr(self, 'reference', None) is None:
            raise RuntimeError('no reference model: call freeze_reference() first')
        with torch.no_grad(), torch.autocast('cuda', dtype=self.compute_dtype, enabled=self.compute_dtype != torch.float32):
            outputs = self.reference(inputs.to(self.device, non_blocking=True).contiguous(memory_format=torch.channels_last))
        return path_log_probs(outputs, paths.to(self.device), self.labelmap)

    def preference_step(self, inputs, paths, criterion, ref_log_probs=None):
        """One training step on preferences: criterion = loss.PreferenceLoss, paths [B, 2, L] (two answers for every image, the preferred first) or, for 2P images of which the
        first P carry the preferred answers, [2P, L].  ref_log_probs None: the frozen reference's.  -> (loss, rewards [P, 2])
        The model runs as it stands and has to be in train mode, as for train_step; the reference runs in eval mode, so the rewards measure the batch's BatchNorm statistics
        against the running ones too."""
        inputs, paths = inputs.to(self.device, non_blocking=True), paths.to(self.device)
        ref = self.reference_log_probs(inputs, paths) if ref_log_probs is None else ref_log_probs.to(self.device)
        return self._feedback_step(inputs, lambda outputs: criterion(outputs, paths, ref))

    def policy_step(self, inputs, paths, advantages, criterion, old_log_probs=None, ref_log_probs=None):
        """One training step on rewards of sampled paths: criterion = loss.ClippedPolicyLoss, paths [B, G, L] or [B, L], advantages [B, G] or [B].  ref_log_probs None: the
        frozen reference's where the criterion has a KL term.  -> (loss, stats [2])
        Paths and old_log_probs are the caller's: nothing here samples.  Modes as in preference_step: ratios start at 1 if old_log_probs come from a train-mode forward of the
        same batch; those of an eval-mode forward differ by its BatchNorm statistics."""
        inputs, paths = inputs.to(self.device, non_blocking=True), paths.to(self.device)
        if ref_log_probs is None and criterion.kl_coef != 0.0:
            ref_log_probs = self.reference_log_probs(inputs, paths)
        at = lambda t: None if t is None else t.to(self.device)
        adv, old, ref = at(advantages), at(old_log_probs), at(ref_log_probs)
        return self._feedback_step(inputs, lambda outputs: criterion(outputs, paths, adv, old, ref))

    def _feedback_step(self, inputs, criterion):
        """train_step with a criterion of the outputs alone that returns (loss, what it reports); the mean is over the LOCAL batch, as there."""
        pend = self.__dict__.setdefault('_steps_in_flight', [])
        if len(pend) >= 2:
            pend.pop(0).synchronize()
        inputs = inputs.to(self.device, non_blocking=True).contiguous(memory_format=torch.channels_last)
        self.arena.zero_grad()
        with torch.autocast('cuda', dtype=self.compute_dtype, enabled=self.compute_dtype != torch.float32):
            outputs = self.model(inputs)
        loss, report = criterion(outputs)
        loss.backward()
        if self.overlap is not None:
            self.overlap.join()
        self.reducer.finish()
        self.arena.adam_step(self.lr, grad_scale=1.0 / self.world)
        done = torch.cuda.Event(); done.record(); pend.append(done)
        return loss.detach(), report
