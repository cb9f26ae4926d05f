"""What a module makes of its weights (concatenations, copies in 8 bits) and keeps from one call to the next."""
import torch


def prepared(owner, name, tag, make):
    """`make()`, a tuple of tensors, kept as `owner.<name>` while `tag` (the weights' versions, places and types) stays the same.

    Any thread and stream may read what is kept: it is finished before another caller can find it (the stream that makes it is
    waited for, once per change of the weights), and its memory waits for every stream that has read it before it is used for
    something else.  Inside a graph's capture nothing is kept, since what is captured is not there before a replay: such a graph
    makes the tensors at each replay, unless a call before the capture has made them."""
    entry = getattr(owner, name)
    if entry is None or entry[0] != tag:
        made = make()
        if made[0].is_cuda:
            with torch.cuda.device(made[0].device):
                if torch.cuda.is_current_stream_capturing():
                    return made
                stream = torch.cuda.current_stream()
                stream.synchronize()
            entry = (tag, made, {stream.cuda_stream})
        else:
            entry = (tag, made, set())
        setattr(owner, name, entry)
    _, made, streams = entry
    if made[0].is_cuda:
        handle = torch._C._cuda_getCurrentRawStream(made[0].device.index)
        if handle not in streams:
            stream = torch.cuda.current_stream(made[0].device)
            for t in made:
                t.record_stream(stream)
            streams.add(handle)
    return made


class Prepares:
    """Mixin of modules that keep such tensors, under the names in `_prepared`: copies and pickles go without, since in another
    process other weights can have the same versions and places."""
    _prepared = ()

    def __getstate__(self):
        return {**self.__dict__, **dict.fromkeys(self._prepared)}

    def __setstate__(self, state):
        super().__setstate__({**state, **dict.fromkeys(self._prepared)})
