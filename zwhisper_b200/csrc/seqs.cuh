// Where the tokens of a call are (zwg_seqs, include/zwgpu.h), read on the device.
#pragma once
#include "common.cuh"
#include "kernels.h"

namespace zwg {

struct Place {
    int past;   // position of the call's token 0
    int count;  // tokens of this sequence in the call; 0: none, or an entry out of range
};

// Sequence b's place; `room` is the number of positions there are. An entry out of range
// leaves the sequence out and sets the error word.
ZWG_DEV Place place_of(const Seqs& s, int b, int room, int* err) {
    Place p{s.n_past, s.n};
    if (s.past) p.past = __ldcg(s.past + b);
    if (s.count) p.count = __ldcg(s.count + b);
    if (p.past < 0 || p.past > s.n_past || p.count < 0 || p.count > s.n || p.count > room - p.past) {
        set_error(err, kErrBounds);
        p.past = p.count = 0;
    }
    return p;
}

}  // namespace zwg
