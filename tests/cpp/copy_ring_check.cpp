// CopyRing (exl3cu_ring.h) against a fake barrier: "<stages> <copies> <the wait that gives up, from 0; -1: none>" prints the
// (slot, parity) of every wait, those of the drain behind a '|'.
#include <cstdio>
#include <cstdlib>

#include "exl3cu_ring.h"

template <unsigned S> void run(int copies, int fails) {
    exl3cu::CopyRing<S> ring;
    int waits = 0, started = 0, used = 0;
    const auto wait = [&](unsigned slot, unsigned parity) {
        std::printf("%u%u ", slot, parity);
        return waits++ != fails;
    };
    for (; started < copies && started < int(S); ++started)
        if (ring.slot(started) != unsigned(started) % S) std::exit(2);
    for (; used < copies; ++used) {
        if (ring.slot() != unsigned(used) % S) std::exit(3);
        if (!ring.next(wait)) break;
        if (started < copies && ring.slot(S - 1) != unsigned(started++) % S) std::exit(4);  // where the last one was
    }
    std::printf("| ");
    ring.drain(started - used, wait);
    std::printf("\n");
}

int main(int argc, char ** argv) {
    if (argc != 4) return 1;
    const int stages = std::atoi(argv[1]), copies = std::atoi(argv[2]), fails = std::atoi(argv[3]);
    if (stages == 2) run<2>(copies, fails);
    else if (stages == 3) run<3>(copies, fails);
    else return 1;
    return 0;
}
